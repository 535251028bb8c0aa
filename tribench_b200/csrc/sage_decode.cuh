// sage_decode.cuh — attention of few query rows per key/value head over the paged cache (single
// generated tokens, drafts of a few tokens).
//
// Per query row of head group h (G query heads share key/value head h): s_j = scale q . K_j over the
// visible keys, o = sum_j softmax(s)_j V_j. Key j < L is visible to the query at position p when
// j <= p (causal) and, with a window W, j > p - W or j < sinks. A row that sees nothing gives 0.
//
// What bounds it: the cache is read once, so HBM (16-bit: 4 D bytes per key and head, INT8: 2 D + 8),
// and for INT8, at half the bytes, the issue slots of widening the codes. The products are
// mma.sync.m16n8k16 with the keys as the 16-row side: S^T = K Q^T and O^T = V^T P^T, so that 8 query
// rows fill a product and the softmax holds 4 scores per lane and 16 keys (a tcgen05 tile's 128 rows
// would be almost all padding). P^T changes sides by movmatrix.
//
// Work split. The unit is a tile of 64 keys of one (sequence, head, tile of 8 NR query rows) item. All
// tiles of the call, in that order, form one line, cut into equal pieces, one per CTA: every CTA
// streams the same number of tiles whatever the lengths are, and the host needs to know none of
// them. A piece that holds an item whole writes its output; an item cut between pieces leaves
// unnormalised partial sums (fp32) in the workspace, which paged_combine_kernel joins in a fixed
// order, so that results do not depend on timing.
//
// CTA: four consumer warps and a producer warp that loads tiles by TMA (one box per page and
// operand) through a ring of stages. Each consumer warp owns 16 of a tile's 64 keys, with its own
// running maximum, sum and output accumulators (registers); the four are joined once per item. K and
// V fragments come from the swizzled tiles by ldmatrix (16-bit), or as plain byte loads widened in
// registers (INT8).
//
// The maximum is lazy: it moves, and the outputs are rescaled, only when a score's logarithm exceeds it
// by more than 8, so most tiles need no reduction over lanes. P <= 2^8 is rounded to the type of the
// cache as an operand of the second product, half a step (bf16 2^-8, fp16 2^-11) of each weight; scores,
// sums and outputs are fp32. Outputs are off from 64 bits by 1.0 to 1.4 times what the rounding of the result
// alone gives.
//
// INT8. K: byte c + 128 zero-extended is the fp16 subnormal (c + 128) 2^-24, exact, without an
// instruction beyond the byte permutation; the scores become 2^24 S' - 128 sum(q), then times k_scale.
// V: codes as exact fp16 values; their weights w_j = p_j v_scale_j are rounded to fp16 in units of 2^E,
// E per query row: 2^E <= the largest w_j that the row has met < 2^(E + 14), so a weight is off by 2^-11
// of itself or 2^-25 of the largest one, whatever the scales of keys that the row does not see or hardly
// attends to. Row maxima of the scores (for the sum) and units (for the outputs) move together, when a
// weight or an exponential outgrows its range. bf16 queries are brought to fp16 by a power of two per
// row: 8 significant bits fit into 11, and what falls below 2^-24 of the row's largest value is lost
// far under bf16's own rounding.
//
// Measured (B200, one token of each of 16 sequences of 20000, 64/8 heads, head_dim 128, calls back to back):
// 16 bit 199 us, 6.58 TB/s, the rate of a plain copy; INT8 118 us, 5.7 TB/s of codes and scales (at 4 sequences
// of 16000, under the profiler, issue slots 45 % busy, DRAM 49 %). Ragged batches pay for the start and the join:
// 64 sequences of 200 to 8192 tokens, 32/8 heads, 16 bit 106 us, 5.6 TB/s. INT8 with 16 rows of an item 171 us (two
// tokens each), with 32, in two items that each stream the cache, 311 us.
#pragma once

#include <type_traits>

#include "sage_paged.cuh"
#include "sm100_ptx.cuh"

namespace sage {

constexpr int kDecWarps = 4;                         // consumer warps
constexpr int kDecThreads = 32 * (kDecWarps + 1);    // + the producer warp
constexpr int kDecKeys = 64;                         // keys per tile
constexpr int kDecMaxRows = 16;                      // query rows per item, at most: 8 NR
constexpr int kDecMaxPieces = 3 * 148;               // CTAs, at most

struct DecodeParams {
  PagedSeqs s;
  const void* q;
  void* o;
  int64_t q_st, q_sh, o_st, o_sh;  // element strides: token, head
  int Hkv, G;
  int page_shift, pages;
  const float* k_scale;            // INT8: [pages][Hkv][page]
  const float* v_scale;
  int causal, window, sinks;       // window 0: none
  float scale_log2;                // sm_scale * log2(e)
  float* part;                     // [2 * CTAs][rows][D] unnormalised outputs
  float* part_ml;                  // [2 * CTAs][rows][4]: max of scores, sum, INT8: E of the outputs' unit 2^(max + E)
  int4* desc;                      // [CTAs]: the item that a CTA's piece begins and does not end (sequence,
                                   // head, query tile or block, pieces that follow with its rest; 0: none)
  // Rows of the chunk kernel's blocks: parts of a head group (1 up to 128 heads), query heads of a
  // part, tokens of a query tile (128 / Gp)
  int parts, Gp, TT;
  unsigned long long wait_limit_ns;
};

template <int D, bool I8, int NR>
struct DecodeCfg {
  static constexpr int ROWS = 8 * NR;
  static constexpr int ELT = I8 ? 1 : 2;
  static constexpr int ROW_BYTES = D * ELT;
  static constexpr int ATOMS = ROW_BYTES > 128 ? 2 : 1;            // 128-byte column atoms per row
  static constexpr int BOX = ROW_BYTES > 128 ? 128 / ELT : D;      // TMA box width, elements
  static constexpr int TILE = kDecKeys * ROW_BYTES;                // K (or V) bytes of a stage
  static constexpr int SCALES = I8 ? 256 : 0;                      // scale bytes of a stage, K or V
  static constexpr int STAGE = 2 * TILE + (I8 ? 1024 : 0);         // tiles start on 1024 bytes
  // CTAs per SM: HBM needs about 45 KB in flight per SM; INT8 also wants warps to issue from
  static constexpr int CTAS = (I8 && NR == 1) ? 3 : 2;
  static constexpr int NS = I8 ? (D == 128 ? 3 : 6) : (D == 128 ? 2 : 4);
  static constexpr int RED_STRIDE = D + 4;                         // floats per row: bank spread
  static constexpr int OFF_RED = NS * STAGE;
  static constexpr int OFF_ML = OFF_RED + kDecWarps * ROWS * RED_STRIDE * 4;
  static constexpr int OFF_BAR = OFF_ML + kDecWarps * ROWS * 4 * 4;
  static constexpr int OFF_MISC = OFF_BAR + 2 * NS * 8;
  static constexpr int OFF_SEG = (OFF_MISC + 56 + 15) / 16 * 16;
  static constexpr int SMEM = 1024 + OFF_SEG + 64;
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "CTAs per SM");
};

// Key tiles of one sequence that some query of it sees: the sinks' tiles, then the rest.
struct TileSpan {
  int ns;      // tiles [0, ns) hold the sinks
  int tw;      // then tiles [tw, tw + count - ns)
  int count;   // at least 1 where the sequence has queries
};
__device__ __forceinline__ TileSpan tile_span(const PagedSeq& q, int window, int sinks, int keys) {
  TileSpan t;
  const int lo = window ? max(0, q.len - q.n - window + 1) : 0;  // first key of the first query's window
  t.ns = window ? (min(sinks, lo) + keys - 1) / keys : 0;
  t.tw = max(lo / keys, t.ns);
  t.count = t.ns + max(0, (q.len + keys - 1) / keys - t.tw);
  if (q.n == 0) t.count = 0;
  else t.count = max(t.count, 1);
  return t;
}
__device__ __forceinline__ int tile_at(const TileSpan& t, int i) { return i < t.ns ? i : t.tw + i - t.ns; }

// One segment of a CTA's piece: tiles [t0, t0 + n) of an item.
struct DecodeSegment {
  PagedSeq sq;
  TileSpan ts;
  int b, h, mt, t0, n, more;
};
static_assert(sizeof(DecodeSegment) <= 64, "DecodeCfg::SMEM");

template <int ROWS>
__device__ __forceinline__ int64_t decode_tiles(const DecodeParams& p, int b) {
  const PagedSeq sq = paged_seq(p.s, b);
  const TileSpan ts = tile_span(sq, p.window, p.sinks, kDecKeys);
  return (int64_t)p.Hkv * ((sq.n * (int64_t)p.G + ROWS - 1) / ROWS) * ts.count;
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Four bytes u = code + 128 of `w` (two's complement codes with the sign bit flipped) as fp16 codes:
// 0x6400 + u is the fp16 value 1024 + u, and subtracting 1152 is exact.
__device__ __forceinline__ uint32_t biased_to_half2(uint32_t bits) {
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&bits), __float2half2_rn(1152.0f));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Transpose of an 8 x 8 matrix of 16-bit values held as mma fragments.
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127
// exponent of |x|, clamped to what pow2 takes either way
__device__ __forceinline__ int exponent(float x) { return min(max((int)((__float_as_uint(x) >> 23) & 255) - 127, -126), 120); }

// INT8: outputs in units of 2^(m + e) (m: maximum of the scores, e: exponent of the weights' unit), seen from a
// maximum ms >= m: the exponent that is sure not to make them larger by 2 or more.
__device__ __forceinline__ float unit_under(float m, float e, float ms) { return fmaxf(e + ceilf(m - ms), -126.0f); }
// No score yet: finite, so that differences of maxima are numbers.
constexpr float kNoScore = -3.402823466e38f;

// T: element type of q, o and a 16-bit cache. NR: query rows of an item / 8.
template <int D, bool I8, typename T, int NR>
__global__ void __launch_bounds__(kDecThreads, DecodeCfg<D, I8, NR>::CTAS)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const DecodeParams p) {
  using C = DecodeCfg<D, I8, NR>;
  using M = typename std::conditional<I8, __half, T>::type;  // operand type of the products
  constexpr int KS = D / 16;   // k-steps of q . K
  constexpr int NT = D / 16;   // 16-channel tiles of the output
  constexpr float LAZY = 8.0f;
  // INT8: the part of the subnormals' 2^24 that goes to the scales of the keys, as 2^24 times a large query's unit
  // would leave fp32
  constexpr float K_UNIT = 1048576.0f;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + C::NS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC);
  int* start_b = reinterpret_cast<int*>(smem + C::OFF_MISC + 4);
  int64_t* start_rem = reinterpret_cast<int64_t*>(smem + C::OFF_MISC + 8);
  int64_t* warp_sum = reinterpret_cast<int64_t*>(smem + C::OFF_MISC + 16);  // [5]
  const int warp = warp_id(), lane = lane_id(), cta = blockIdx.x;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::NS; ++s) {
      mbar_init(full + s, I8 ? 33 : 1);  // INT8: the producer's lanes bring four scales each
      mbar_init(empty + s, kDecWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  // This CTA's piece of the line of tiles: each thread adds up the tiles of a run of sequences.
  const int run = (p.s.batch + kDecThreads - 1) / kDecThreads;
  const int b_lo = min(p.s.batch, (int)threadIdx.x * run), b_hi = min(p.s.batch, b_lo + run);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += decode_tiles<C::ROWS>(p, b);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kDecWarps + 1; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const int64_t per = (total + gridDim.x - 1) / gridDim.x;
  const int64_t begin = per * cta;
  const int64_t count = min(per, total - begin);  // tiles of this CTA
  if (count <= 0) {  // uniform
    if (threadIdx.x == 0) p.desc[cta] = make_int4(0, 0, 0, 0);
    return;
  }
  if (begin >= before + incl - mine && begin < before + incl) {
    int64_t at = before + incl - mine;
    int b = b_lo;
    for (; b < b_hi - 1; ++b) {
      const int64_t t = decode_tiles<C::ROWS>(p, b);
      if (begin < at + t) break;
      at += t;
    }
    *start_b = b;
    *start_rem = begin - at;
  }
  __syncthreads();

  int b = *start_b;
  int64_t rem = *start_rem;  // tiles of sequence b before this piece
  int64_t left = count;

  if (warp == kDecWarps) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const int page = 1 << p.page_shift;
    const int rows = min(page, kDecKeys);            // rows of a box
    const int ppt = kDecKeys / rows;                 // pages of a tile
    const int batch_tiles = 32 / ppt;                // tiles whose page numbers the 32 lanes hold
    const int boxes = ppt * 2 * C::ATOMS;
    int it = 0;
    bool ok = true;
    while (left > 0 && ok && b < p.s.batch) {
      const PagedSeq sq = paged_seq(p.s, b);
      const TileSpan ts = tile_span(sq, p.window, p.sinks, kDecKeys);
      const int nmt = (sq.n * p.G + C::ROWS - 1) / C::ROWS;
      const int64_t all = (int64_t)p.Hkv * nmt * ts.count;
      if (rem >= all) { rem = 0; ++b; continue; }  // the next sequence with tiles
      const int item = (int)(rem / ts.count), t0 = (int)(rem - (int64_t)item * ts.count);
      const int h = item / nmt;
      const int n = (int)min((int64_t)(ts.count - t0), left);
      const int* table = p.s.table + (int64_t)b * p.s.table_stride;
      auto page_of = [&](int i) {  // this lane's page of tiles [i, i + batch_tiles)
        const int ti = i + lane / ppt;
        if (ti >= t0 + n) return -1;
        const int pg = ((tile_at(ts, ti) * kDecKeys) >> p.page_shift) + lane % ppt;
        return pg < p.s.width ? table[pg] : -1;
      };
      int next = page_of(t0);
      for (int i0 = t0; i0 < t0 + n && ok; i0 += batch_tiles) {
        const int ids = next;
        if (i0 + batch_tiles < t0 + n) next = page_of(i0 + batch_tiles);
        const int i1 = min(t0 + n, i0 + batch_tiles);
        for (int i = i0; i < i1; ++i, ++it) {
          const int s = it % C::NS;
          if (it >= C::NS) {
            ok = mbar_wait(empty + s, ((it / C::NS) - 1) & 1, abort_flag, 1, p.wait_limit_ns);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
          uint8_t* st = smem + s * C::STAGE;
          if (lane == 0)
            mbar_arrive_expect_tx(full + s, 2 * C::TILE);
          __syncwarp();
          // box l: sub-page, then column atom, then K / V
          const int sub = lane % ppt;
          const int id = __shfl_sync(0xffffffffu, ids, (i - i0) * ppt + sub);
          const int y = (tile_at(ts, i) * kDecKeys) & (page - 1);  // 0 where a tile holds whole pages
          const int rest = lane / ppt, atom = rest % C::ATOMS, isv = rest / C::ATOMS;
          if (lane < boxes)
            tma_load_4d(st + isv * C::TILE + atom * (kDecKeys * 128) + sub * rows * (C::ROW_BYTES > 128 ? 128 : C::ROW_BYTES),
                        isv ? &tmV : &tmK, full + s, atom * C::BOX, y, h, id);
          if constexpr (I8) {
            // scales of keys 4 x .. 4 x + 3, K's from lanes 0-15, V's from 16-31: a copy of 16 bytes
            // each costs less than a box per page
            const int x = (lane & 15) * 4, sv = lane >> 4;
            const int pg = __shfl_sync(0xffffffffu, ids, (i - i0) * ppt + x / rows);
            const bool in = pg >= 0 && pg < p.pages;
            const float* src = (sv ? p.v_scale : p.k_scale) +
                               (in ? ((((int64_t)pg * p.Hkv + h) << p.page_shift) + ((y + x) & (page - 1))) : 0);
            cp_async16(smem_u32(st + 2 * C::TILE + sv * C::SCALES) + x * 4, src, in);
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full + s)) : "memory");
          }
        }
      }
      rem += n;
      left -= n;
    }
    // The last copies must have landed before the block's shared memory goes, whoever gave up meanwhile (the
    // abort flag does not end these waits, their limit does).
    for (int j = max(0, it - C::NS); j < it; ++j) {
      volatile int none = 0;
      (void)mbar_wait(full + j % C::NS, (j / C::NS) & 1, &none, 1, p.wait_limit_ns);
    }
    return;
  }

  // ------------------------------------------------------------ consumers
  const int g = lane >> 2, t = lane & 3;  // fragment row / column group
  float* red = reinterpret_cast<float*>(smem + C::OFF_RED);
  float* ml = reinterpret_cast<float*>(smem + C::OFF_ML);
  const uint32_t smem_base = smem_u32(smem);
  int it = 0;
  bool ok = true;
  int4 cut = make_int4(0, 0, 0, 0);  // the item that this piece begins and does not end
  DecodeSegment& seg = *reinterpret_cast<DecodeSegment*>(smem + C::OFF_SEG);
  for (;;) {
    // One thread finds the segment for all: the warps meet at barriers, so they must agree on it even
    // if the arrays change under a running call.
    if (threadIdx.x == 0) {
      seg.more = 0;
      for (; left > 0 && b < p.s.batch; ++b, rem = 0) {
        const PagedSeq sq = paged_seq(p.s, b);
        const TileSpan ts = tile_span(sq, p.window, p.sinks, kDecKeys);
        const int nmt = (sq.n * p.G + C::ROWS - 1) / C::ROWS;
        if (rem >= (int64_t)p.Hkv * nmt * ts.count) continue;
        const int item = (int)(rem / ts.count), t0 = (int)(rem - (int64_t)item * ts.count), h = item / nmt;
        const int n = (int)min((int64_t)(ts.count - t0), left);
        seg = DecodeSegment{sq, ts, b, h, item - h * nmt, t0, n, 1};
        rem += n;
        left -= n;
        break;
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kDecWarps * 32) : "memory");
    if (!seg.more) break;
    const PagedSeq sq = seg.sq;
    const TileSpan ts = seg.ts;
    const int h = seg.h, mt = seg.mt, t0 = seg.t0, n = seg.n;
    const int rows = min(C::ROWS, sq.n * p.G - mt * C::ROWS);  // valid rows of the item
    const int first = sq.len - sq.n;                           // position of the first new token
    // This thread's query rows 8 nt + 2 t, 8 nt + 2 t + 1: the keys [lo, hi) (and [0, sinks)) that they see
    int lo[NR][2], hi[NR][2];
#pragma unroll
    for (int nt = 0; nt < NR; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int pos = first + (mt * C::ROWS + min(8 * nt + 2 * t + c, rows - 1)) / p.G;
        hi[nt][c] = p.causal ? pos + 1 : sq.len;
        lo[nt][c] = p.window ? pos - p.window + 1 : 0;
      }
    // bounds over all rows of the item: keys no row sees, and tiles that every row sees whole
    const int tok_a = mt * C::ROWS / p.G, tok_b = (mt * C::ROWS + rows - 1) / p.G;
    const int any_hi = p.causal ? first + tok_b + 1 : sq.len, all_hi = p.causal ? first + tok_a + 1 : sq.len;
    const int any_lo = p.window ? first + tok_a - p.window + 1 : 0, all_lo = p.window ? first + tok_b - p.window + 1 : 0;

    // Q fragments: row 8 nt + g. 16-bit: k index = channel. INT8: lane column t holds channels
    // [t D/4, (t + 1) D/4), k-step s its channels 4 s .. 4 s + 3, so that a K row's codes are contiguous
    // per lane.
    uint32_t qf[NR][KS][2];
    float qa[NR][2], qb[NR][2];  // score = qa S + qb, of this thread's rows 2 t, 2 t + 1
#pragma unroll
    for (int nt = 0; nt < NR; ++nt) {
      const int row = 8 * nt + g, fr = mt * C::ROWS + row, tok = fr / p.G, hd = fr - tok * p.G;
      const bool in = row < rows;
      const T* qp = static_cast<const T*>(p.q) + (in ? (int64_t)(sq.base + tok) * p.q_st + (int64_t)(h * p.G + hd) * p.q_sh : 0);
      if constexpr (!I8) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            qf[nt][s][half] = in ? *reinterpret_cast<const uint32_t*>(qp + s * 16 + half * 8 + t * 2) : 0u;
        qa[nt][0] = qa[nt][1] = p.scale_log2;
        qb[nt][0] = qb[nt][1] = 0.0f;
      } else {
        float unit = 1.0f, sum = 0.0f;
        uint4 raw[D / 32];
        uint32_t m = 0;
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          raw[x] = in ? ldg_nc_v4(qp + t * (D / 4) + x * 8) : make_uint4(0u, 0u, 0u, 0u);
          if constexpr (!std::is_same<T, __half>::value) {
            float f[8];
            Half8<T>::to_float(raw[x], f);
#pragma unroll
            for (int y = 0; y < 8; ++y) m = max(m, abs_bits(f[y]));
          }
        }
        if constexpr (!std::is_same<T, __half>::value) {
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
          unit = pow2(exponent(__uint_as_float(m)));
        }
        const float down = 1.0f / unit;  // a power of two: exact
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          float f[8];
          Half8<T>::to_float(raw[x], f);
          if constexpr (!std::is_same<T, __half>::value) {
#pragma unroll
            for (int y = 0; y < 8; ++y) f[y] *= down;
            raw[x] = Half8<__half>::from_float(f);
            Half8<__half>::to_float(raw[x], f);
          }
          sum += ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
          qf[nt][2 * x][0] = raw[x].x;
          qf[nt][2 * x][1] = raw[x].y;
          qf[nt][2 * x + 1][0] = raw[x].z;
          qf[nt][2 * x + 1][1] = raw[x].w;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const float a = p.scale_log2 * unit;
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // row 2 t + c is that of lanes 4 (2 t + c)
          const float ar = __shfl_sync(0xffffffffu, a, 4 * (2 * t + c)), sr = __shfl_sync(0xffffffffu, sum, 4 * (2 * t + c));
          qa[nt][c] = ar * (16777216.0f / K_UNIT);
          qb[nt][c] = (-128.0f / K_UNIT * sr) * ar;
        }
      }
    }

    float acc[NT][NR][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int nt = 0; nt < NR; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][nt][c] = 0.0f;
    float m1[NR][2], l[NR][2];  // l: this lane's part
#pragma unroll
    for (int nt = 0; nt < NR; ++nt) {
      m1[nt][0] = m1[nt][1] = I8 ? kNoScore : -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
    }
    int unit[NR][2];    // INT8: weights are in units of 2^unit, down = 2^-unit
    float down[NR][2];
#pragma unroll
    for (int nt = 0; nt < NR; ++nt) {
      unit[nt][0] = unit[nt][1] = -126;
      down[nt][0] = down[nt][1] = pow2(126);
    }

#pragma unroll 1
    for (int i = t0; i < t0 + n; ++i, ++it) {
      const int s = it % C::NS;
      if (ok) ok = mbar_wait(full + s, (it / C::NS) & 1, abort_flag, 4, p.wait_limit_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) continue;
      const uint32_t kt = smem_base + s * C::STAGE, vt = kt + C::TILE;
      const int key0 = tile_at(ts, i) * kDecKeys;
      const int k_warp = warp * 16;  // this warp's keys of the tile
      // ---- scores of 16 keys x 8 NR rows; this lane: keys g, g + 8
      float sc[NR][4];
#pragma unroll
      for (int nt = 0; nt < NR; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[nt][c] = 0.0f;
      float vs[2] = {1.0f, 1.0f};
      if constexpr (!I8) {
        const int r = lane & 7, mi = lane >> 3;
        const int key = k_warp + (mi & 1) * 8 + r;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int chunk = 2 * ks + (mi >> 1);
          uint32_t a[4];
          ldmatrix_x4(a, kt + (chunk >> 3) * (kDecKeys * 128) + key * 128 + (((chunk & 7) ^ r) << 4));
#pragma unroll
          for (int nt = 0; nt < NR; ++nt) mma16816<M>(sc[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NR; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[nt][c] *= qa[nt][c & 1];
      } else {
        uint32_t w[2][D / 16];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int key = k_warp + x * 8 + g;
#pragma unroll
          for (int y = 0; y < D / 64; ++y) {
            const int chunk = t * (D / 64) + y;
            const int sw = D == 128 ? (chunk ^ (key & 7)) : (chunk ^ ((key >> 1) & 3));
            const uint4 v = *reinterpret_cast<const uint4*>(smem + s * C::STAGE + key * D + sw * 16);
            w[x][4 * y] = v.x; w[x][4 * y + 1] = v.y; w[x][4 * y + 2] = v.z; w[x][4 * y + 3] = v.w;
          }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint32_t u0 = w[0][ks] ^ 0x80808080u, u1 = w[1][ks] ^ 0x80808080u;
          const uint32_t a[4] = {__byte_perm(u0, 0u, 0x4140), __byte_perm(u1, 0u, 0x4140), __byte_perm(u0, 0u, 0x4342),
                                 __byte_perm(u1, 0u, 0x4342)};
#pragma unroll
          for (int nt = 0; nt < NR; ++nt) mma16816<M>(sc[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
        }
        const float* scales = reinterpret_cast<const float*>(smem + s * C::STAGE + 2 * C::TILE);
        const int at = k_warp + g;
        // an infinite scale (of a row that holds an infinity) becomes NaN: its codes are 0, but what is left of
        // 2^24 S' - 128 sum(q) after rounding would give it a sign
        float ks0 = scales[at], ks1 = scales[at + 8];
        ks0 = fmaf(ks0, K_UNIT, ks0 - ks0);
        ks1 = fmaf(ks1, K_UNIT, ks1 - ks1);
        vs[0] = scales[C::SCALES / 4 + at];
        vs[1] = scales[C::SCALES / 4 + at + 8];
#pragma unroll
        for (int nt = 0; nt < NR; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[nt][c] = fmaf(sc[nt][c], qa[nt][c & 1], qb[nt][c & 1]) * (c < 2 ? ks0 : ks1);
      }
      // ---- mask
      const bool whole = key0 + kDecKeys <= all_hi && (key0 >= all_lo || key0 + kDecKeys <= p.sinks);
      uint32_t vm[2] = {0xffffffffu, 0xffffffffu};  // 16-bit: V rows 2 t (+ 1), + 8 that some query sees
      uint32_t seen = 0xffffffffu;                  // bit 4 nt + c
      if (!whole) {
        seen = 0;
#pragma unroll
        for (int nt = 0; nt < NR; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int key = key0 + k_warp + (c >> 1) * 8 + g;
            const bool see = key < hi[nt][c & 1] && (key >= lo[nt][c & 1] || key < p.sinks);
            if (!see) sc[nt][c] = -INFINITY;
            seen |= see ? 1u << (4 * nt + c) : 0u;
          }
        if constexpr (!I8) {
          // rows that no query sees may hold anything (an unused page's NaN): 0 instead, as their weight is
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int key = key0 + k_warp + x * 8 + 2 * t;
            const bool a = key < any_hi && (key >= any_lo || key < p.sinks);
            const bool z = key + 1 < any_hi && (key + 1 >= any_lo || key + 1 < p.sinks);
            vm[x] = (a ? 0xffffu : 0u) | (z ? 0xffff0000u : 0u);
          }
        } else {
#pragma unroll
          for (int x = 0; x < 2; ++x) {  // nor may an unused scale
            const int key = key0 + k_warp + x * 8 + g;
            if (!(key < any_hi && (key >= any_lo || key < p.sinks))) vs[x] = 0.0f;
          }
        }
      }
      uint32_t pf[NR][2];  // weights, as the B operand of O^T = V^T P^T
      if constexpr (!I8) {
        // ---- the maximum, where a score outgrew it
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NR; ++nt)
          grow |= fmaxf(sc[nt][0], sc[nt][2]) > m1[nt][0] + LAZY || fmaxf(sc[nt][1], sc[nt][3]) > m1[nt][1] + LAZY;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nt = 0; nt < NR; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = fmaxf(sc[nt][c], sc[nt][c + 2]);
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
              const float mn = fmaxf(m1[nt][c], mx);
              const float alpha = mn == -INFINITY ? 1.0f : ex2_approx(m1[nt][c] - mn);
              m1[nt][c] = mn;
              l[nt][c] *= alpha;
#pragma unroll
              for (int x = 0; x < NT; ++x) {
                acc[x][nt][c] *= alpha;
                acc[x][nt][c + 2] *= alpha;
              }
            }
        }
        // ---- weights
#pragma unroll
        for (int nt = 0; nt < NR; ++nt) {
          const float u0 = m1[nt][0] == -INFINITY ? 0.0f : m1[nt][0], u1 = m1[nt][1] == -INFINITY ? 0.0f : m1[nt][1];
          const float e[4] = {ex2_approx(sc[nt][0] - u0), ex2_approx(sc[nt][1] - u1), ex2_approx(sc[nt][2] - u0),
                              ex2_approx(sc[nt][3] - u1)};
          l[nt][0] += e[0] + e[2];
          l[nt][1] += e[1] + e[3];
          pf[nt][0] = movmatrix(pack2<M>(e[0], e[1]));
          pf[nt][1] = movmatrix(pack2<M>(e[2], e[3]));
        }
      } else {
        // ---- exponentials and weights; where one outgrew its range, new maxima and units, and once more
        float e[NR][4], w8[NR][4];
        auto weigh = [&] {
          bool grow = false;
#pragma unroll
          for (int nt = 0; nt < NR; ++nt) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float2 a = fadd2(make_float2(sc[nt][2 * x], sc[nt][2 * x + 1]), make_float2(-m1[nt][0], -m1[nt][1]));
              const float2 y = make_float2(ex2_approx(a.x), ex2_approx(a.y));
              const float2 z = fmul2(fmul2(y, make_float2(vs[x], vs[x])), make_float2(down[nt][0], down[nt][1]));
              e[nt][2 * x] = y.x; e[nt][2 * x + 1] = y.y;
              w8[nt][2 * x] = z.x; w8[nt][2 * x + 1] = z.y;
            }
            if (!whole) {
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if (!((seen >> (4 * nt + c)) & 1u)) w8[nt][c] = 0.0f;  // the scale may be a NaN
            }
            grow |= fmax3(fmaxf(fabsf(w8[nt][0]), fabsf(w8[nt][1])), fabsf(w8[nt][2]), fabsf(w8[nt][3])) > 16384.0f ||
                    fmax3(fmaxf(e[nt][0], e[nt][1]), e[nt][2], e[nt][3]) > 1.152921504606847e18f;  // 2^60
          }
          return grow;
        };
        if (__builtin_expect(__any_sync(0xffffffffu, weigh()), 0)) {
#pragma unroll
          for (int nt = 0; nt < NR; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = fmaxf(sc[nt][c], sc[nt][c + 2]);
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
              const float mo = m1[nt][c], mn = fmaxf(mo, mx);
              // fmaxf drops a NaN (of a scale that this row does not see: 0 * NaN)
              float top = fmaxf(fmaxf(fabsf(ex2_approx(sc[nt][c] - mn) * vs[0]), fabsf(ex2_approx(sc[nt][c + 2] - mn) * vs[1])), 0.0f);
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
              // the weights of before have shrunk by 2^(mn - mo), so may their unit
              const int before = mo == kNoScore ? -126 : unit[nt][c] - (int)ceilf(fminf(mn - mo, 256.0f));
              const int now = max(max(exponent(top), before), -126);
              const float alpha = ex2_approx(mo - mn), move = ex2_approx((mo - mn) + (float)(unit[nt][c] - now));
              m1[nt][c] = mn;
              unit[nt][c] = now;
              down[nt][c] = pow2(-now);
              l[nt][c] *= alpha;
#pragma unroll
              for (int x = 0; x < NT; ++x) {
                acc[x][nt][c] *= move;
                acc[x][nt][c + 2] *= move;
              }
            }
          (void)weigh();
        }
#pragma unroll
        for (int nt = 0; nt < NR; ++nt) {
          const float2 sum = fadd2(make_float2(l[nt][0], l[nt][1]), fadd2(make_float2(e[nt][0], e[nt][1]), make_float2(e[nt][2], e[nt][3])));
          l[nt][0] = sum.x;
          l[nt][1] = sum.y;
          pf[nt][0] = movmatrix(pack2<M>(w8[nt][0], w8[nt][1]));
          pf[nt][1] = movmatrix(pack2<M>(w8[nt][2], w8[nt][3]));
        }
      }
      // ---- O^T += V^T P^T over this warp's 16 keys
      if constexpr (!I8) {
        const int r = lane & 7, mi = lane >> 3;
        const int key = k_warp + (mi >> 1) * 8 + r;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int chunk = 2 * j + (mi & 1);
          uint32_t a[4];
          ldmatrix_x4_trans(a, vt + (chunk >> 3) * (kDecKeys * 128) + key * 128 + (((chunk & 7) ^ r) << 4));
          a[0] &= vm[0]; a[1] &= vm[0]; a[2] &= vm[1]; a[3] &= vm[1];
#pragma unroll
          for (int nt = 0; nt < NR; ++nt) mma16816<M>(acc[j][nt], a, pf[nt][0], pf[nt][1]);
        }
      } else {
        // rows g and g + 8 of output tile i are channels g D/8 + 2 i and + 1: a lane's D/8 codes of a key
        // are contiguous
        constexpr int W = D / 32;  // words of codes per key
        uint32_t w[4][W];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int key = k_warp + 2 * t + (x & 1) + (x >> 1) * 8;
          const uint8_t* base = smem + s * C::STAGE + C::TILE + key * D;
          if constexpr (D == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(base + ((g ^ (key & 7)) << 4));
            w[x][0] = v.x; w[x][1] = v.y; w[x][2] = v.z; w[x][3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(base + ((((g >> 1) ^ ((key >> 1) & 3)) << 4) | ((g & 1) << 3)));
            w[x][0] = v.x; w[x][1] = v.y;
          }
#pragma unroll
          for (int y = 0; y < W; ++y) w[x][y] ^= 0x80808080u;
        }
#pragma unroll
        for (int y = 0; y < W; ++y) {
          // bytes of keys 2t, 2t + 1 interleaved, channel by channel; the same for 2t + 8, 2t + 9
          const uint32_t k01 = __byte_perm(w[0][y], w[1][y], 0x5140), k23 = __byte_perm(w[0][y], w[1][y], 0x7362);
          const uint32_t n01 = __byte_perm(w[2][y], w[3][y], 0x5140), n23 = __byte_perm(w[2][y], w[3][y], 0x7362);
          const uint32_t a[4] = {biased_to_half2(__byte_perm(k01, 0x64646464u, 0x4140)), biased_to_half2(__byte_perm(k01, 0x64646464u, 0x4342)),
                                 biased_to_half2(__byte_perm(n01, 0x64646464u, 0x4140)), biased_to_half2(__byte_perm(n01, 0x64646464u, 0x4342))};
          const uint32_t z[4] = {biased_to_half2(__byte_perm(k23, 0x64646464u, 0x4140)), biased_to_half2(__byte_perm(k23, 0x64646464u, 0x4342)),
                                 biased_to_half2(__byte_perm(n23, 0x64646464u, 0x4140)), biased_to_half2(__byte_perm(n23, 0x64646464u, 0x4342))};
#pragma unroll
          for (int nt = 0; nt < NR; ++nt) {
            mma16816<M>(acc[2 * y][nt], a, pf[nt][0], pf[nt][1]);
            mma16816<M>(acc[2 * y + 1][nt], z, pf[nt][0], pf[nt][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + s);
    }

    // ---- join the four warps: maxima, sums and units first
#pragma unroll
    for (int nt = 0; nt < NR; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], o);
        if (g == 0) {
          float* x = ml + (warp * C::ROWS + 8 * nt + 2 * t + c) * 4;
          x[0] = m1[nt][c];
          x[1] = l[nt][c];
          if constexpr (I8) x[2] = (float)unit[nt][c];
        }
      }
    asm volatile("bar.sync 1, %0;" ::"n"(kDecWarps * 32) : "memory");
#pragma unroll
    for (int nt = 0; nt < NR; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = 8 * nt + 2 * t + c;
        float ms = I8 ? kNoScore : -INFINITY, f;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) ms = fmaxf(ms, ml[(w * C::ROWS + row) * 4]);
        if constexpr (I8) {
          float eo = -126.0f;
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w)
            eo = fmaxf(eo, unit_under(ml[(w * C::ROWS + row) * 4], ml[(w * C::ROWS + row) * 4 + 2], ms));
          f = ex2_approx((m1[nt][c] - ms) + ((float)unit[nt][c] - eo));
        } else {
          f = ex2_approx(m1[nt][c] - (ms == -INFINITY ? 0.0f : ms));
        }
        float* dst = red + (warp * C::ROWS + row) * C::RED_STRIDE;
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          if constexpr (!I8) {
            dst[16 * x + g] = acc[x][nt][c] * f;
            dst[16 * x + g + 8] = acc[x][nt][c + 2] * f;
          } else {
            *reinterpret_cast<float2*>(dst + g * (D / 8) + 2 * x) = make_float2(acc[x][nt][c] * f, acc[x][nt][c + 2] * f);
          }
        }
      }
    asm volatile("bar.sync 1, %0;" ::"n"(kDecWarps * 32) : "memory");
    const bool begins = t0 == 0, ends = t0 + n == ts.count;
    const int slot = 2 * cta + (begins ? 1 : 0);
#pragma unroll 1
    for (int idx = threadIdx.x; idx < C::ROWS * (D / 4); idx += kDecWarps * 32) {
      const int row = idx / (D / 4), c4 = idx % (D / 4);
      if (row >= rows) continue;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float ms = I8 ? kNoScore : -INFINITY, eo = -126.0f, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(red + (w * C::ROWS + row) * C::RED_STRIDE + c4 * 4);
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
        ms = fmaxf(ms, ml[(w * C::ROWS + row) * 4]);
      }
      const float use = ms == -INFINITY ? 0.0f : ms;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        const float* y = ml + (w * C::ROWS + row) * 4;
        sum = fmaf(y[1], ex2_approx(y[0] - use), sum);
        if constexpr (I8) eo = fmaxf(eo, unit_under(y[0], y[2], ms));
      }
      if (begins && ends) {
        const float inv = sum == 0.0f ? 0.0f : (I8 ? pow2((int)eo) : 1.0f) / sum;
        const int fr = mt * C::ROWS + row, tok = fr / p.G, hd = fr - tok * p.G;
        T* dst = static_cast<T*>(p.o) + (int64_t)(sq.base + tok) * p.o_st + (int64_t)(h * p.G + hd) * p.o_sh + c4 * 4;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
      } else {
        *reinterpret_cast<float4*>(p.part + ((int64_t)slot * C::ROWS + row) * D + c4 * 4) = o;
        if (c4 == 0) *reinterpret_cast<float4*>(p.part_ml + (slot * C::ROWS + row) * 4) = make_float4(ms, sum, I8 ? eo : 0.0f, 0.0f);
      }
    }
    if (begins && !ends) cut = make_int4(seg.b, h, mt, (int)((ts.count - n + per - 1) / per));
    asm volatile("bar.sync 1, %0;" ::"n"(kDecWarps * 32) : "memory");
  }
  if (threadIdx.x == 0) p.desc[cta] = cut;
}

// Joins the pieces of items that the pieces' borders cut: the item that piece c begins without ending
// (slot 2 c + 1) has its other parts in slots 2 c' of the pieces that follow. Block (c, row) joins one
// row: eight warps share its parts, lanes hold D / 32 channels each.
constexpr int kCombineThreads = 256;
template <int D, bool I8, typename T, int NR>
__global__ void __launch_bounds__(kCombineThreads) paged_combine_kernel(const DecodeParams p) {
  constexpr int E = D / 32, W = kCombineThreads / 32, ROWS = 8 * NR;
  __shared__ float s_o[W][D];
  __shared__ float s_ml[W][3];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 d = p.desc[blockIdx.x];
  if (d.w == 0) return;
  const int warp = warp_id(), lane = lane_id(), row = blockIdx.y;
  const PagedSeq sq = paged_seq(p.s, d.x);
  const int fr = d.z * ROWS + row;
  if (fr >= sq.n * p.G) return;
  const int tok = fr / p.G, hd = fr - tok * p.G;
  // eo: INT8, the outputs are in units of 2^(ms + eo)
  float o[E], ms = I8 ? kNoScore : -INFINITY, l = 0.0f, eo = -126.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll 4
  for (int j = warp; j <= d.w; j += W) {
    const int64_t slot = j == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + j);
    const float4 x = *reinterpret_cast<const float4*>(p.part_ml + (slot * ROWS + row) * 4);
    const float* src = p.part + (slot * ROWS + row) * D + lane * E;
    float v[E];
    if constexpr (E == 4) {
      const float4 y = *reinterpret_cast<const float4*>(src);
      v[0] = y.x; v[1] = y.y; v[2] = y.z; v[3] = y.w;
    } else {
      const float2 y = *reinterpret_cast<const float2*>(src);
      v[0] = y.x; v[1] = y.y;
    }
    const float mn = fmaxf(ms, x.x), us = mn == -INFINITY ? 0.0f : mn;
    float fa = ex2_approx(ms - us), fb = ex2_approx(x.x - us);
    l = fmaf(l, fa, x.y * fb);
    if constexpr (I8) {
      const float en = fmaxf(unit_under(ms, eo, mn), unit_under(x.x, x.z, mn));
      fa = ex2_approx((ms - mn) + (eo - en));
      fb = ex2_approx((x.x - mn) + (x.z - en));
      eo = en;
    }
    ms = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], fa, v[e] * fb);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
  if (lane == 0) {
    s_ml[warp][0] = ms;
    s_ml[warp][1] = l;
    s_ml[warp][2] = eo;
  }
  __syncthreads();
  if (warp != 0) return;
  ms = I8 ? kNoScore : -INFINITY;
  eo = -126.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) ms = fmaxf(ms, s_ml[w][0]);
  if constexpr (I8) {
#pragma unroll
    for (int w = 0; w < W; ++w) eo = fmaxf(eo, unit_under(s_ml[w][0], s_ml[w][2], ms));
  }
  l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
  const float us = ms == -INFINITY ? 0.0f : ms;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    float f = ex2_approx(s_ml[w][0] - us);
    l = fmaf(s_ml[w][1], f, l);
    if constexpr (I8) f = ex2_approx((s_ml[w][0] - ms) + (s_ml[w][2] - eo));
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(s_o[w][lane * E + e], f, o[e]);
  }
  const float inv = l == 0.0f ? 0.0f : (I8 ? pow2((int)eo) : 1.0f) / l;
  T* dst = static_cast<T*>(p.o) + (int64_t)(sq.base + tok) * p.o_st + (int64_t)(d.y * p.G + hd) * p.o_sh + lane * E;
  if constexpr (E == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack2<T>(o[0] * inv, o[1] * inv);
}

}  // namespace sage
