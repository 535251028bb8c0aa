// sage_chunk.cuh — attention of many query rows per key/value head over the paged cache (chunks of
// new prompt tokens, whole prompts, mixed batches) on the tensor cores.
//
// The mathematics is that of sage_decode.cuh; with 256 query rows per tile of keys the products bound
// it (4 D operations per pair), and behind them the softmax's issue slots, as in sage_attn.cuh, whose
// pipeline this is: two 128-row query tiles, S = Q K^T and O += P V as tcgen05.mma into TMEM, one
// softmax warpgroup per query tile, MMA issued by one thread.
//
// Rows. The rows of one key/value head are the (token, query head of the group) pairs in that order:
// row r of a sequence is token r / G, head r % G. A block of 256 rows then covers 256 / G tokens, all
// query heads of the group sharing every tile of keys, and a short chunk of G heads still fills rows.
//
// Work split. Blocks of one sequence need different numbers of key tiles (causal mask, window). A
// one-block kernel (paged_schedule_kernel) lists the blocks with their tiles and cuts the line of all
// tiles (block by block, head by head) into equal pieces, one per SM; each CTA runs through its piece
// segment by segment, the tile ring running on across segments. A block cut between pieces leaves
// fp32 partial sums, joined afterwards in a fixed order, as in sage_decode.cuh.
//
// Warps: 0-7 softmax (two warpgroups), 8 TMA producer, 9 MMA issuer, 10-11 helpers, which bring the
// next segment's query rows in with cp.async as soon as its last Q K^T has run, and put zeros over rows
// of V that no query sees (an unused row may hold a NaN, which its weight of 0 would not silence).
#pragma once

#include "sage_attn.cuh"
#include "sage_decode.cuh"

namespace sage {

constexpr int kChunkRows = 256;     // query rows per block
constexpr int kChunkPieces = 148;   // CTAs: one per SM
constexpr int kChunkThreads = 384;

// One block of query rows: the sequence's span, the block's number and its key tiles.
struct ChunkItem {
  int base, n, len, b;
  int blk, ns, tw, count;
};
struct ChunkPiece {
  int item, head, tile, count;  // where it starts, tiles
};

struct ChunkParams {
  DecodeParams d;
  ChunkItem* items;
  int64_t* prefix;      // [items + 1] tiles of one head before an item (schedule only)
  ChunkPiece* pieces;   // [kChunkPieces]
  int* per;             // tiles of a piece
  int max_items;
};

template <int D, typename T>
struct ChunkCfg {
  static constexpr bool PRE_BIAS = false, QK_F16 = true, PV_FP8 = false;
  static constexpr int BM = 128, BN = 128;
  static constexpr int NS = (D == 128) ? 2 : 4;  // K/V ring stages
  static constexpr int TILE = 128 * D * 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * TILE;
  static constexpr int OFF_V = OFF_K + NS * TILE;
  static constexpr int OFF_BAR = OFF_V + NS * TILE;
  static constexpr int NUM_BARS = 2 + 4 * NS + 12;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int SMEM_BYTES = 1024 + OFF_MISC + 64;
  static_assert(SMEM_BYTES <= 227 * 1024 && SMEM_BYTES > 114 * 1024, "one CTA per SM");
  static constexpr int REGS_SOFTMAX = 216, REGS_OTHER = 72;  // as in AttnCfg
  static constexpr uint32_t QK_LAYOUT = kLayoutSW128, QK_SBO = 1024;
  static constexpr int QK_STEPS = D / 16;
  static __device__ __forceinline__ uint32_t qk_step_offset(int kk, int rows) {
    return (32 * kk / 128) * rows * 128 + (32 * kk) % 128;
  }
  static constexpr int ATOMS = D / 64;  // 128-byte column atoms
  static constexpr uint32_t V_LBO = BN * 128, V_SBO = 1024;
  static constexpr bool SEP_P = (D == 64);
  static constexpr uint32_t P_COL = SEP_P ? 128 + D : 64;
  static constexpr uint32_t FMT = std::is_same<T, __half>::value ? kFmtF16 : kFmtBF16;
  static constexpr uint32_t IDESC_QK = make_idesc(kFmtD_F32, FMT, FMT, 0, 0, BM, BN);
  static constexpr uint32_t IDESC_PV = make_idesc(kFmtD_F32, FMT, FMT, 0, 1, BM, D);
  static constexpr float LAZY = 8.0f;
  static constexpr int EMU = 12;
};

// ------------------------------------------------------------------ schedule
__device__ __forceinline__ int chunk_blocks(const PagedSeq& sq, int G) {
  return (sq.n * G + kChunkRows - 1) / kChunkRows;
}

// The tiles of 128 keys that block `blk` of a sequence needs.
__device__ __forceinline__ void chunk_tiles(const ChunkParams& p, const PagedSeq& sq, int blk, ChunkItem* it) {
  const int G = p.d.G;
  const int tok_a = blk * kChunkRows / G, tok_b = min(sq.n * G, (blk + 1) * kChunkRows) - 1;
  const int last = tok_b / G, first = sq.len - sq.n;
  const int lo = p.d.window ? max(0, first + tok_a - p.d.window + 1) : 0;
  const int hi = p.d.causal ? first + last + 1 : sq.len;
  it->ns = p.d.window ? min((min(p.d.sinks, lo) + 127) / 128, (max(hi, 0) + 127) / 128) : 0;
  it->tw = max(lo / 128, it->ns);
  it->count = max(1, it->ns + max(0, (hi + 127) / 128 - it->tw));
}

constexpr int kScheduleThreads = 1024;
__global__ void __launch_bounds__(kScheduleThreads) paged_schedule_kernel(const ChunkParams p) {
  __shared__ int64_t s_warp[32];
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
    int64_t w = s_warp[lane];
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
    const int nb = chunk_blocks(sq, p.d.G);
    int64_t total = 0;
    const int64_t at = n_items + block_scan(nb, &total);
    for (int l = 0; l < 32; ++l) {
      PagedSeq q;
      q.base = __shfl_sync(0xffffffffu, sq.base, l);
      q.n = __shfl_sync(0xffffffffu, sq.n, l);
      q.len = __shfl_sync(0xffffffffu, sq.len, l);
      const int64_t off = __shfl_sync(0xffffffffu, at, l);
      const int blocks = chunk_blocks(q, p.d.G);
      for (int k = lane; k < blocks; k += 32) {
        if (off + k >= p.max_items) break;  // the host's bound holds for any prefix sums; kept as a fence
        ChunkItem it;
        it.base = q.base; it.n = q.n; it.len = q.len; it.b = b0 + warp * 32 + l;
        it.blk = k;
        chunk_tiles(p, q, k, &it);
        p.items[off + k] = it;
      }
    }
    n_items += total;
  }
  if (n_items > p.max_items) n_items = p.max_items;
  __syncthreads();
  // ---- tiles before each block
  int64_t tiles = 0;
  for (int64_t i0 = 0; i0 < n_items; i0 += kScheduleThreads) {
    const int64_t i = i0 + tid;
    int64_t total = 0;
    const int64_t at = tiles + block_scan(i < n_items ? p.items[i].count : 0, &total);
    if (i < n_items) p.prefix[i] = at;
    tiles += total;
  }
  __syncthreads();
  // ---- equal pieces of the line
  const int64_t all = tiles * p.d.Hkv;
  const int64_t per = max((all + kChunkPieces - 1) / kChunkPieces, (int64_t)1);
  if (tid == 0) *p.per = (int)per;
  if (tid < kChunkPieces) {
    ChunkPiece c{0, 0, 0, 0};
    const int64_t begin = per * tid;
    if (begin < all) {
      // the last block whose line position is <= begin
      int64_t lo = 0, n = n_items;
      while (n > 1) {
        const int64_t half = n / 2;
        if (p.prefix[lo + half] * p.d.Hkv <= begin) { lo += half; n -= half; }
        else n = half;
      }
      const int64_t rem = begin - p.prefix[lo] * p.d.Hkv;
      const int cnt = p.items[lo].count;
      c.item = (int)lo;
      c.head = (int)(rem / cnt);
      c.tile = (int)(rem % cnt);
      c.count = (int)min(per, all - begin);
    }
    p.pieces[tid] = c;
  }
}

// ------------------------------------------------------------------ attention
// One segment of a CTA's piece: tiles [t0, t0 + n) of a block for one head.
struct ChunkWalk {
  const ChunkItem* items;
  int item, head, tile, left, Hkv;
  ChunkItem it;
  int n;
  __device__ __forceinline__ ChunkWalk(const ChunkParams& p, int cta) {
    const ChunkPiece c = p.pieces[cta];
    items = p.items;
    item = c.item; head = c.head; tile = c.tile; left = c.count;
    Hkv = p.d.Hkv;
    if (left > 0) load();
  }
  __device__ __forceinline__ void load() {
    const int4 a = reinterpret_cast<const int4*>(items + item)[0], z = reinterpret_cast<const int4*>(items + item)[1];
    it.base = a.x; it.n = a.y; it.len = a.z; it.b = a.w;
    it.blk = z.x; it.ns = z.y; it.tw = z.z; it.count = z.w;
    n = min(it.count - tile, left);
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next() {
    left -= n;
    tile = 0;
    if (++head == Hkv) {
      head = 0;
      ++item;
      if (left > 0) load();
    } else {
      n = min(it.count, left);
    }
  }
  __device__ __forceinline__ int rows(int G) const { return min(kChunkRows, it.n * G - it.blk * kChunkRows); }
  __device__ __forceinline__ int key0(int j) const {  // first key of tile `tile + j`
    const int i = tile + j;
    return (i < it.ns ? i : it.tw + i - it.ns) * 128;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

template <int D, typename T>
__global__ void __launch_bounds__(kChunkThreads, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const ChunkParams cp) {
  using C = ChunkCfg<D, T>;
  const DecodeParams& p = cp.d;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar_q = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* bar_qfree = bar_q + 1;
  uint64_t* bar_vraw = bar_q + 2;  // [stage]: V landed, rows that no query sees still to be cleared
  uint64_t* bar_kfull = bar_vraw + C::NS;
  uint64_t* bar_vfull = bar_kfull + C::NS;
  uint64_t* bar_kvempty = bar_vfull + C::NS;
  uint64_t* bar_sfull = bar_kvempty + C::NS;
  uint64_t* bar_phalf = bar_sfull + 2;
  uint64_t* bar_pfull = bar_phalf + 2;
  uint64_t* bar_odone = bar_pfull + 2;
  uint64_t* bar_sload = bar_odone + 2;
  uint64_t* bar_pvdone = bar_sload + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  const uint32_t warp = warp_id(), lane = lane_id();
  const int cta = blockIdx.x;

  if (threadIdx.x == 0) {
    mbar_init(bar_q, 64);  // the helpers' threads
    mbar_init(bar_qfree, 1);
    for (int s = 0; s < C::NS; ++s) {
      mbar_init(bar_vraw + s, 1);
      mbar_init(bar_kfull + s, 1);
      mbar_init(bar_vfull + s, 1);
      mbar_init(bar_kvempty + s, 1);
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
  ChunkWalk w(cp, cta);
  const int G = p.G;

  // a tile that holds rows of V which no query of the block sees
  auto ragged = [&](int key0) {
    const int first = w.it.len - w.it.n, tok_a = w.it.blk * kChunkRows / G;
    const int tok_b = (w.it.blk * kChunkRows + w.rows(G) - 1) / G;
    const int hi = p.causal ? first + tok_b + 1 : w.it.len;
    const int lo = p.window ? first + tok_a - p.window + 1 : 0;
    return key0 + 128 > hi || (key0 < lo && key0 + 128 > p.sinks);
  };

  if (warp >= 8) {
    regs_dec<C::REGS_OTHER>();
    if (warp == 8) {
      // ------------------------------------------------------------ TMA producer
      const int page = 1 << p.page_shift;
      const int rows = min(page, 128), ppt = 128 / rows;    // rows of a box, pages of a tile
      const int batch_tiles = 32 / ppt;
      const int boxes = ppt * C::ATOMS;                      // of K, and of V
      int it = 0;
      bool ok = true;
      for (; w.more() && ok; w.next()) {
        const int* table = p.s.table + (int64_t)w.it.b * p.s.table_stride;
        auto page_of = [&](int j) {  // this lane's page of tiles [j, j + batch_tiles) of the segment
          const int tj = j + (int)lane / ppt;
          if (tj >= w.n) return -1;
          const int pg = (w.key0(tj) >> p.page_shift) + (int)lane % ppt;
          return pg < p.s.width ? table[pg] : -1;
        };
        int next = page_of(0);
        for (int j0 = 0; j0 < w.n && ok; j0 += batch_tiles) {
          const int ids = next;
          if (j0 + batch_tiles < w.n) next = page_of(j0 + batch_tiles);
          const int j1 = min(w.n, j0 + batch_tiles);
          for (int j = j0; j < j1; ++j, ++it) {
            const int s = it % C::NS;
            if (it >= C::NS) {
              ok = mbar_wait(bar_kvempty + s, ((it / C::NS) - 1) & 1, abort_flag, kDevTimeoutProducer, p.wait_limit_ns);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
            }
            const int key0 = w.key0(j);
            uint64_t* vbar = (ragged(key0) ? bar_vraw : bar_vfull) + s;
            if (lane == 0) {
              mbar_arrive_expect_tx(bar_kfull + s, C::TILE);
              mbar_arrive_expect_tx(vbar, C::TILE);
            }
            __syncwarp();
            const int y = key0 & (page - 1);
            for (int x = lane; x < (2 * boxes + 31) / 32 * 32; x += 32) {
              const int sub = x % ppt, rest = x / ppt, atom = rest % C::ATOMS, isv = rest / C::ATOMS;
              const int id = __shfl_sync(0xffffffffu, ids, (j - j0) * ppt + sub);
              if (x < 2 * boxes)
                tma_load_4d(smem + (isv ? C::OFF_V : C::OFF_K) + s * C::TILE + atom * (128 * 128) + sub * rows * 128,
                            isv ? &tmV : &tmK, isv ? vbar : bar_kfull + s, atom * 64, y, w.head, id);
            }
          }
        }
      }
      if (!ok) {  // gave up: wait (bounded) for the copies of K in flight (those of V were issued with them)
        for (int j = max(0, it - C::NS); j < it; ++j) {
          volatile int none = 0;
          (void)mbar_wait(bar_kfull + j % C::NS, (j / C::NS) & 1, &none, kDevTimeoutProducer, p.wait_limit_ns);
        }
      }
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
          const int nt = w.rows(G) > 128 ? 2 : 1, n = w.n;
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
              if (j + 2 == n && t + 1 == nt) umma_commit(bar_qfree);  // the block's queries have been read
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
            if (ok) umma_commit(bar_kvempty + s);
          }
          it0 += n;
          ct0[0] += n;
          if (nt == 2) ct0[1] += n;
        }
      }
    } else {
      // ------------------------------------------------------------ helpers: queries, rows of V nobody sees
      const int hl = (warp - 10) * 32 + lane;
      int it = 0, seg = 0;
      uint32_t raw_phase = 0;  // bit s: phase of bar_vraw[s]
      bool ok = true;
      for (; w.more() && ok; w.next(), ++seg) {
        if (seg > 0) ok = mbar_wait(bar_qfree, (seg - 1) & 1, abort_flag, kDevTimeoutProducer, p.wait_limit_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        constexpr int PR = D / 8;  // 16-byte pieces per row
        const int rows = w.rows(G), fr0 = w.it.blk * kChunkRows;
        const int need = (rows > 128 ? 256 : 128) * PR;
        const char* q = static_cast<const char*>(p.q);
        const uint32_t q_addr = smem_u32(smem + C::OFF_Q);
#pragma unroll 4
        for (int x = hl; x < need; x += 64) {
          const int row = x / PR, c = x % PR, r = row & 127;
          const int fr = fr0 + min(row, rows - 1), tok = fr / G, hd = fr - tok * G;
          cp_async16(q_addr + (row >> 7) * C::TILE + (c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                     q + ((int64_t)(w.it.base + tok) * p.q_st + (int64_t)(w.head * G + hd) * p.q_sh + c * 8) * 2, row < rows);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        mbar_arrive(bar_q);
        const int first = w.it.len - w.it.n, tok_a = fr0 / G, tok_b = (fr0 + rows - 1) / G;
        const int hi = p.causal ? first + tok_b + 1 : w.it.len;
        const int lo = p.window ? first + tok_a - p.window + 1 : 0;
        if (warp == 10) continue;
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
    if (warp == 9) {
      asm volatile("bar.sync 2, %0;" ::"n"(kChunkThreads) : "memory");
      tc_fence_after();
      tmem_dealloc(tmem_base, 512);
    } else {
      asm volatile("bar.arrive 2, %0;" ::"n"(kChunkThreads) : "memory");
    }
  } else {
    // ------------------------------------------------------------ softmax warpgroups
    regs_inc<C::REGS_SOFTMAX>();
    const int t = warp / 4;
    const int row_in_tile = (warp % 4) * 32 + lane;
    const uint32_t lane_base = ((warp % 4) * 32u) << 16;
    const uint32_t s_tmem = tmem_base + lane_base + 256 * t;
    const uint32_t o_tmem = s_tmem + 128;
    int ct = 0, segs = 0;  // tiles and segments of this query tile so far
    bool ok = true;
    int4 cut = make_int4(0, 0, 0, 0);
    for (; w.more() && ok; w.next()) {
      const int rows = w.rows(G);
      if (w.tile == 0 && w.n < w.it.count) {
        const int per = *cp.per;
        cut = make_int4(w.it.b, w.head, w.it.blk, (w.it.count - w.n + per - 1) / per);
      }
      if (t * 128 >= rows) continue;  // no rows in this query tile (uniform over the warpgroup)
      const int n = w.n;
      const int row = t * 128 + row_in_tile, fr = w.it.blk * kChunkRows + min(row, rows - 1);
      const int tok = fr / G, hd = fr - tok * G;
      const int first = w.it.len - w.it.n, pos = first + tok;
      const int hi = p.causal ? pos + 1 : w.it.len;        // this row sees keys [lo, hi) and those of [0, sinks) below hi
      const int lo = p.window ? pos - p.window + 1 : 0;
      // over the rows of this query tile
      const int ta = (w.it.blk * kChunkRows + t * 128) / G, tb = (w.it.blk * kChunkRows + min(rows, t * 128 + 128) - 1) / G;
      const int all_hi = p.causal ? first + ta + 1 : w.it.len, all_lo = p.window ? first + tb - p.window + 1 : 0;
      float m_run = -INFINITY, l_run = 0.0f;
      for (int j = 0; j < n; ++j) {
        if (!__all_sync(0xffffffffu, mbar_wait(bar_sfull + t, (ct + j) & 1, abort_flag, kDevTimeoutSoftmax, p.wait_limit_ns))) { ok = false; break; }
        tc_fence_after();
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
        const int key0 = w.key0(j);
        const int up = hi - key0, down = lo - key0, sk = p.sinks - key0;
        const bool masked = key0 + 128 > all_hi || (key0 < all_lo && key0 + 128 > p.sinks);
        if (masked) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= up || (c < down && c >= sk)) b[c] = -INFINITY;
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
        const float tmax = fmaxf(hm[0], hm[1]) * p.scale_log2;
        const bool upd = tmax > m_run + C::LAZY;
        const float m_new = upd ? tmax : m_run;
        const float alpha = upd ? ex2_approx(m_run - m_new) : 1.0f;
        const bool rescale = j > 0 && __any_sync(0xffffffffu, upd);
        const float m_use = (m_new == -INFINITY) ? 0.0f : m_new;
        const float2 scv = make_float2(p.scale_log2, p.scale_log2), ccv = make_float2(-m_use, -m_use);
        float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
          uint32_t pk[32];
#pragma unroll
          for (int pr = 0; pr < 32; ++pr) {
            const int c = h2 * 64 + 2 * pr;
            const float2 a = ffma2(make_float2(b[c], b[c + 1]), scv, ccv);
            float2 e;
            if ((c % 32) >= 32 - C::EMU) {
              e = exp2_poly2(a);
            } else {
              e.x = ex2_approx(a.x);
              e.y = ex2_approx(a.y);
            }
            acc[pr & 3] = fadd2(acc[pr & 3], e);
            pk[pr] = pack2<T>(e.x, e.y);
          }
          // the polynomial's least result, 2^-125, is no zero in bf16
          if (std::is_same<T, __nv_bfloat16>::value && masked) {
#pragma unroll
            for (int pr = 0; pr < 32; ++pr) {
              const int c = h2 * 64 + 2 * pr;
              if (c >= up || (c < down && c >= sk)) pk[pr] &= 0xffff0000u;
              if (c + 1 >= up || (c + 1 < down && c + 1 >= sk)) pk[pr] &= 0xffffu;
            }
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
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += 32) {
              uint32_t orow[32];
              tmem_ld32_sync(o_tmem + c0, orow);
#pragma unroll
              for (int c = 0; c < 32; ++c) orow[c] = __float_as_uint(__uint_as_float(orow[c]) * alpha);
              tmem_st32(o_tmem + c0, orow);
            }
          }
        }
        if (!ok) break;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar_pfull + t);
        const float2 s01 = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
        l_run = fmaf(l_run, alpha, s01.x + s01.y);
        m_run = m_new;
      }
      if (!ok) break;
      if (!__all_sync(0xffffffffu, mbar_wait(bar_odone + t, segs & 1, abort_flag, kDevTimeoutEpilogue, p.wait_limit_ns))) { ok = false; break; }
      tc_fence_after();
      ct += n;
      ++segs;
      const bool whole = w.tile == 0 && n == w.it.count;
      const float inv = whole ? (m_run == -INFINITY ? 0.0f : 1.0f / l_run) : 1.0f;
      const int64_t slot = 2 * cta + (w.tile == 0 ? 1 : 0);
      T* dst = static_cast<T*>(p.o) + (int64_t)(w.it.base + tok) * p.o_st + (int64_t)(w.head * G + hd) * p.o_sh;
      float* part = p.part + (slot * kChunkRows + row) * D;
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t orow[32];
        tmem_ld32_sync(o_tmem + c0, orow);
        if (row < rows) {
          if (whole) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              float f[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(orow[8 * v + e]) * inv;
              *reinterpret_cast<uint4*>(dst + c0 + 8 * v) = Half8<T>::from_float(f);
            }
          } else {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<uint4*>(part + c0 + 4 * v) = make_uint4(orow[4 * v], orow[4 * v + 1], orow[4 * v + 2], orow[4 * v + 3]);
          }
        }
      }
      if (!whole && row < rows)
        *reinterpret_cast<float4*>(p.part_ml + (slot * kChunkRows + row) * 4) = make_float4(m_run, l_run, m_run, 0.0f);
      tc_fence_before();
    }
    if (threadIdx.x == 0) p.desc[cta] = cut;
    tc_fence_before();
    asm volatile("bar.arrive 2, %0;" ::"n"(kChunkThreads) : "memory");
  }
}

}  // namespace sage
