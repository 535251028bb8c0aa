// sage_decode.cuh — attention of few query rows per key/value head over the paged cache (single
// generated tokens, drafts of a few tokens).
//
// Per query row of head group h (G query heads share key/value head h): s_j = scale q . K_j over the
// visible keys, o = sum_j softmax(s)_j V_j. Key j < L is visible to the query at position p when
// j <= p (causal) and, with a window W, j > p - W or j < sinks. A row that sees nothing gives 0.
//
// What bounds it: the cache is read once, so HBM (16-bit: 4 D bytes per key and head, INT8: 2 D + 8);
// the products are 16-row mma.sync tiles, whose rate no shape here comes near to needing
// (a 128-row tcgen05 tile would be almost all padding).
//
// Work split. The unit is a tile of 64 keys of one (sequence, head, 16-row query tile) item. All
// tiles of the call, in that order, form one line, cut into equal pieces, one per CTA: every CTA
// streams the same number of tiles whatever the lengths are, and the host needs to know none of
// them. A piece that holds an item whole writes its output; an item cut between pieces leaves
// unnormalised partial sums (fp32) in the workspace, which paged_combine_kernel joins in a fixed
// order, so that results do not depend on timing.
//
// CTA: four consumer warps and a producer warp that loads tiles by TMA (one box per page and
// operand) through a ring of stages. Each consumer warp owns 16 of a tile's 64 keys, with its own
// running maximum, sum and output accumulators (registers); the four are joined once per item. K and
// V fragments come from the swizzled tiles by ldmatrix (16-bit), or as plain byte loads converted in
// registers (INT8: the codes are exact in fp16).
//
// INT8: scores are (q . code) * k_scale; the weights of V's codes are p_j v_scale_j, kept relative to
// their own running maximum, since v_scale may be anything while fp16 may not. bf16 queries are
// brought to fp16 by a power of two per row: 8 significant bits fit into 11, and what falls below
// 2^-24 of the row's largest value is lost far under bf16's own rounding.
#pragma once

#include <type_traits>

#include "sage_paged.cuh"
#include "sm100_ptx.cuh"

namespace sage {

constexpr int kDecWarps = 4;                         // consumer warps
constexpr int kDecThreads = 32 * (kDecWarps + 1);    // + the producer warp
constexpr int kDecKeys = 64;                         // keys per tile
constexpr int kDecRows = 16;                         // query rows per item
constexpr int kDecPieces = 2 * 148;                  // CTAs: two per SM

struct DecodeParams {
  PagedSeqs s;
  const void* q;
  void* o;
  int64_t q_st, q_sh, o_st, o_sh;  // element strides: token, head
  int Hkv, G;
  int page_shift;
  int causal, window, sinks;       // window 0: none
  float scale_log2;                // sm_scale * log2(e)
  float* part;                     // [2 * CTAs][16][D] unnormalised outputs
  float* part_ml;                  // [2 * CTAs][16][4]: max of scores, sum, max of weights
  int4* desc;                      // [CTAs]: the item that a CTA's piece begins and does not end (sequence,
                                   // head, query tile or block, pieces that follow with its rest; 0: none)
  // Rows of the chunk kernel's blocks: parts of a head group (1 up to 128 heads), query heads of a
  // part, tokens of a query tile (128 / Gp)
  int parts, Gp, TT;
  unsigned long long wait_limit_ns;
};

template <int D, bool I8>
struct DecodeCfg {
  static constexpr int ELT = I8 ? 1 : 2;
  static constexpr int ROW_BYTES = D * ELT;
  static constexpr int ATOMS = ROW_BYTES > 128 ? 2 : 1;            // 128-byte column atoms per row
  static constexpr int BOX = ROW_BYTES > 128 ? 128 / ELT : D;      // TMA box width, elements
  static constexpr int TILE = kDecKeys * ROW_BYTES;                // K (or V) bytes of a stage
  static constexpr int SCALES = I8 ? 512 : 0;                      // scale bytes of a stage, K or V
  static constexpr int STAGE = 2 * TILE + 2 * SCALES;
  // Ring: 64 KB in flight per CTA, two CTAs per SM (what HBM needs in flight is about 45 KB per SM)
  static constexpr int NS = 65536 / (2 * TILE) > 6 ? 6 : 65536 / (2 * TILE);
  static constexpr int RED_STRIDE = D + 8;                         // floats per row: bank spread
  static constexpr int OFF_RED = NS * STAGE;
  static constexpr int OFF_ML = OFF_RED + kDecWarps * kDecRows * RED_STRIDE * 4;
  static constexpr int OFF_BAR = OFF_ML + kDecWarps * kDecRows * 4 * 4;
  static constexpr int OFF_MISC = OFF_BAR + 2 * NS * 8;
  static constexpr int SMEM = 1024 + OFF_MISC + 64;
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

__device__ __forceinline__ int64_t decode_tiles(const DecodeParams& p, int b) {
  const PagedSeq sq = paged_seq(p.s, b);
  const TileSpan ts = tile_span(sq, p.window, p.sinks, kDecKeys);
  return (int64_t)p.Hkv * ((sq.n * (int64_t)p.G + kDecRows - 1) / kDecRows) * ts.count;
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

// T: element type of q, o and a 16-bit cache.
template <int D, bool I8, typename T>
__global__ void __launch_bounds__(kDecThreads, 2)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const __grid_constant__ CUtensorMap tmKs, const __grid_constant__ CUtensorMap tmVs,
                        const DecodeParams p) {
  using C = DecodeCfg<D, I8>;
  using M = typename std::conditional<I8, __half, T>::type;  // operand type of the products
  constexpr int KS = D / 16;   // k-steps of q . K
  constexpr int NT = D / 8;    // 8-column tiles of the output
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
      mbar_init(full + s, 1);
      mbar_init(empty + s, kDecWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  // This CTA's piece of the line of tiles: each thread adds up the tiles of a run of sequences.
  const int run = (p.s.batch + kDecThreads - 1) / kDecThreads;
  const int b_lo = min(p.s.batch, (int)threadIdx.x * run), b_hi = min(p.s.batch, b_lo + run);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += decode_tiles(p, b);
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
      const int64_t t = decode_tiles(p, b);
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
    const int boxes = ppt * 2 * C::ATOMS + (I8 ? ppt * 2 : 0);
    int it = 0;
    bool ok = true;
    while (left > 0 && ok && b < p.s.batch) {
      const PagedSeq sq = paged_seq(p.s, b);
      const TileSpan ts = tile_span(sq, p.window, p.sinks, kDecKeys);
      const int nmt = (sq.n * p.G + kDecRows - 1) / kDecRows;
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
            mbar_arrive_expect_tx(full + s, 2 * C::TILE + (I8 ? 2 * kDecKeys * 4 : 0));
          __syncwarp();
          // box l: sub-page, then column atom, then K / V (then the scales)
          const int sub = lane % ppt;
          const int id = __shfl_sync(0xffffffffu, ids, (i - i0) * ppt + sub);
          const int y = (tile_at(ts, i) * kDecKeys) & (page - 1);  // 0 where a tile holds whole pages
          const int rest = lane / ppt;
          if (lane < boxes) {
            if (rest < 2 * C::ATOMS) {
              const int atom = rest % C::ATOMS, isv = rest / C::ATOMS;
              tma_load_4d(st + isv * C::TILE + atom * (kDecKeys * 128) + sub * rows * (C::ROW_BYTES > 128 ? 128 : C::ROW_BYTES),
                          isv ? &tmV : &tmK, full + s, atom * C::BOX, y, h, id);
            } else {
              const int isv = rest - 2 * C::ATOMS;
              tma_load_4d(st + 2 * C::TILE + isv * C::SCALES + sub * 128, isv ? &tmVs : &tmKs, full + s, y, h, id, 0);
            }
          }
        }
      }
      rem += n;
      left -= n;
    }
    if (!ok) {
      // gave up: wait (bounded) for the copies in flight before the block's shared memory goes
      for (int j = max(0, it - C::NS); j < it; ++j) {
        volatile int none = 0;
        (void)mbar_wait(full + j % C::NS, (j / C::NS) & 1, &none, 1, p.wait_limit_ns);
      }
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
  while (left > 0 && b < p.s.batch) {
    const PagedSeq sq = paged_seq(p.s, b);
    const TileSpan ts = tile_span(sq, p.window, p.sinks, kDecKeys);
    const int nmt = (sq.n * p.G + kDecRows - 1) / kDecRows;
    const int64_t all = (int64_t)p.Hkv * nmt * ts.count;
    if (rem >= all) { rem = 0; ++b; continue; }
    const int item = (int)(rem / ts.count), t0 = (int)(rem - (int64_t)item * ts.count);
    const int h = item / nmt, mt = item - h * nmt;
    const int n = (int)min((int64_t)(ts.count - t0), left);
    const int rows = min(kDecRows, sq.n * p.G - mt * kDecRows);  // valid rows of the item
    const int first = sq.len - sq.n;                            // position of the first new token
    // this thread's two rows: token and keys [lo, hi) (and [0, sinks)) that it sees
    int lo[2], hi[2];
    const T* qp[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + 8 * r, fr = mt * kDecRows + min(row, rows - 1);
      const int tok = fr / p.G, hd = fr - tok * p.G;
      const int pos = first + tok;
      hi[r] = p.causal ? pos + 1 : sq.len;
      lo[r] = p.window ? pos - p.window + 1 : 0;
      qp[r] = row < rows ? static_cast<const T*>(p.q) + (int64_t)(sq.base + tok) * p.q_st +
                               (int64_t)(h * p.G + hd) * p.q_sh
                         : nullptr;
    }
    // bounds over all rows of the item: keys no row sees, and tiles that every row sees whole
    const int tok_a = mt * kDecRows / p.G, tok_b = (mt * kDecRows + rows - 1) / p.G;
    const int any_hi = p.causal ? first + tok_b + 1 : sq.len, all_hi = p.causal ? first + tok_a + 1 : sq.len;
    const int any_lo = p.window ? first + tok_a - p.window + 1 : 0, all_lo = p.window ? first + tok_b - p.window + 1 : 0;

    // Q fragments. 16-bit: k index = channel. INT8: lane column t holds channels [t D/4, (t+1) D/4),
    // k-step s its channels 4 s .. 4 s + 3, so that a K row's codes are contiguous per lane.
    uint32_t qf[KS][4];
    float qscale[2] = {p.scale_log2, p.scale_log2};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (!I8) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            qf[s][half * 2 + r] =
                qp[r] ? *reinterpret_cast<const uint32_t*>(qp[r] + s * 16 + half * 8 + t * 2) : 0u;
      } else {
        uint4 raw[D / 32];
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
          raw[x] = qp[r] ? ldg_nc_v4(qp[r] + t * (D / 4) + x * 8) : make_uint4(0u, 0u, 0u, 0u);
        if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            qf[2 * x][r] = raw[x].x;
            qf[2 * x][2 + r] = raw[x].y;
            qf[2 * x + 1][r] = raw[x].z;
            qf[2 * x + 1][2 + r] = raw[x].w;
          }
        } else {
          float f[D / 4];
          float m = 0.0f;
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            float e[8];
            Half8<T>::to_float(raw[x], e);
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              f[x * 8 + y] = e[y];
              m = fmaxf(m, fabsf(e[y]));
            }
          }
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          // 2^e <= m < 2^(e+1): multiply by 2^-e, and the scores by 2^e (two factors: e may be -126)
          const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -126), 126);
          const float down = __uint_as_float((uint32_t)(127 - e) << 23);
          qscale[r] *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            const float* y = f + x * 8;
            qf[2 * x][r] = pack2<__half>(y[0] * down, y[1] * down);
            qf[2 * x][2 + r] = pack2<__half>(y[2] * down, y[3] * down);
            qf[2 * x + 1][r] = pack2<__half>(y[4] * down, y[5] * down);
            qf[2 * x + 1][2 + r] = pack2<__half>(y[6] * down, y[7] * down);
          }
        }
      }
    }

    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][c] = 0.0f;
    float m1[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float m2[2] = {-INFINITY, -INFINITY};  // INT8: maximum of score + log2(v_scale)

    for (int i = t0; i < t0 + n; ++i, ++it) {
      const int s = it % C::NS;
      if (ok) ok = mbar_wait(full + s, (it / C::NS) & 1, abort_flag, 4, p.wait_limit_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) continue;
      const uint32_t kt = smem_base + s * C::STAGE, vt = kt + C::TILE;
      const int key0 = tile_at(ts, i) * kDecKeys;
      const int k_warp = warp * 16;  // this warp's keys of the tile
      // ---- scores of 16 rows x 16 keys
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      float lv[2][2] = {{0.f, 0.f}, {0.f, 0.f}};  // INT8: log2(v_scale) of this thread's keys
      if constexpr (!I8) {
        const int r = lane & 7, mi = lane >> 3;
        const int key = k_warp + (mi >> 1) * 8 + r;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int chunk = 2 * ks + (mi & 1);
          uint32_t bf[4];
          ldmatrix_x4(bf, kt + (chunk >> 3) * (kDecKeys * 128) + key * 128 + (((chunk & 7) ^ r) << 4));
          mma16816<M>(sc[0], qf[ks], bf[0], bf[1]);
          mma16816<M>(sc[1], qf[ks], bf[2], bf[3]);
        }
      } else {
        const float* kscale = reinterpret_cast<const float*>(smem + s * C::STAGE + 2 * C::TILE);
        const float* vscale = kscale + C::SCALES / 4;
        float ksc[2][2];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const int key = k_warp + nt * 8 + g;
          uint32_t w[D / 16];
#pragma unroll
          for (int x = 0; x < D / 64; ++x) {
            const int chunk = t * (D / 64) + x;
            const int sw = D == 128 ? (chunk ^ (key & 7)) : (chunk ^ ((key >> 1) & 3));
            const uint4 v = *reinterpret_cast<const uint4*>(smem + s * C::STAGE + key * D + sw * 16);
            w[4 * x] = v.x; w[4 * x + 1] = v.y; w[4 * x + 2] = v.z; w[4 * x + 3] = v.w;
          }
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const uint32_t u = w[ks] ^ 0x80808080u;
            mma16816<M>(sc[nt], qf[ks], biased_to_half2(__byte_perm(u, 0x64646464u, 0x4140)),
                        biased_to_half2(__byte_perm(u, 0x64646464u, 0x4342)));
          }
          // a page's scales start on 128 bytes
          const int kk = k_warp + nt * 8 + 2 * t;
          const int sh = min(p.page_shift, 6);
          const int at = (kk >> sh) * (sh < 5 ? 32 : (1 << sh)) + (kk & ((1 << sh) - 1));
          const float2 k2 = *reinterpret_cast<const float2*>(kscale + at);
          const float2 v2 = *reinterpret_cast<const float2*>(vscale + at);
          ksc[nt][0] = k2.x; ksc[nt][1] = k2.y;
          lv[nt][0] = __log2f(v2.x); lv[nt][1] = __log2f(v2.y);
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[nt][c] *= ksc[nt][c & 1];
      }
      // ---- mask and softmax
      const bool whole = key0 + kDecKeys <= all_hi && (key0 >= all_lo || key0 + kDecKeys <= p.sinks);
      float w2[2][4];  // INT8: exponents of the weights
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = c >> 1, key = key0 + k_warp + nt * 8 + 2 * t + (c & 1);
          const bool see = whole || (key < hi[r] && (key >= lo[r] || key < p.sinks));
          const float x = sc[nt][c] * qscale[r];
          sc[nt][c] = see ? x : -INFINITY;
          if constexpr (I8) w2[nt][c] = see ? x + lv[nt][c & 1] : -INFINITY;
        }
      uint32_t pf[4];
      float p_out[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m1[r], mx), use = mn == -INFINITY ? 0.0f : mn;
        const float alpha = ex2_approx(m1[r] - use);
        m1[r] = mn;
        float sum = 0.0f;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float e = ex2_approx(sc[nt][2 * r + c] - use);
            sum += e;
            p_out[nt][2 * r + c] = e;
          }
        l[r] = fmaf(l[r], alpha, sum);
        float beta = alpha;
        if constexpr (I8) {
          float my = fmaxf(fmaxf(w2[0][2 * r], w2[0][2 * r + 1]), fmaxf(w2[1][2 * r], w2[1][2 * r + 1]));
          my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 1));
          my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 2));
          const float wn = fmaxf(m2[r], my), uw = wn == -INFINITY ? 0.0f : wn;
          beta = ex2_approx(m2[r] - uw);
          m2[r] = wn;
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) p_out[nt][2 * r + c] = ex2_approx(w2[nt][2 * r + c] - uw);
        }
        if (__any_sync(0xffffffffu, beta != 1.0f)) {
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            acc[x][2 * r] *= beta;
            acc[x][2 * r + 1] *= beta;
          }
        }
      }
      pf[0] = pack2<M>(p_out[0][0], p_out[0][1]);
      pf[1] = pack2<M>(p_out[0][2], p_out[0][3]);
      pf[2] = pack2<M>(p_out[1][0], p_out[1][1]);
      pf[3] = pack2<M>(p_out[1][2], p_out[1][3]);
      // ---- P . V over this warp's 16 keys
      if constexpr (!I8) {
        // rows that no query sees may hold anything (an unused page's NaN): 0 instead, as their weight is
        uint32_t vm[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int key = key0 + k_warp + x * 8 + 2 * t;
          const bool a = whole || (key < any_hi && (key >= any_lo || key < p.sinks));
          const bool z = whole || (key + 1 < any_hi && (key + 1 >= any_lo || key + 1 < p.sinks));
          vm[x] = (a ? 0xffffu : 0u) | (z ? 0xffff0000u : 0u);
        }
        const int r = lane & 7, mi = lane >> 3;
        const int key = k_warp + (mi & 1) * 8 + r;
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
          const int chunk = 2 * j + (mi >> 1);
          uint32_t bf[4];
          ldmatrix_x4_trans(bf, vt + (chunk >> 3) * (kDecKeys * 128) + key * 128 + (((chunk & 7) ^ r) << 4));
          mma16816<M>(acc[2 * j], pf, bf[0] & vm[0], bf[1] & vm[1]);
          mma16816<M>(acc[2 * j + 1], pf, bf[2] & vm[0], bf[3] & vm[1]);
        }
      } else {
        // column n of output tile i is channel n D/8 + i: a lane's D/8 codes of a key are contiguous
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
          const uint32_t a01 = __byte_perm(w[0][y], w[1][y], 0x5140), a23 = __byte_perm(w[0][y], w[1][y], 0x7362);
          const uint32_t c01 = __byte_perm(w[2][y], w[3][y], 0x5140), c23 = __byte_perm(w[2][y], w[3][y], 0x7362);
          mma16816<M>(acc[4 * y], pf, biased_to_half2(__byte_perm(a01, 0x64646464u, 0x4140)),
                      biased_to_half2(__byte_perm(c01, 0x64646464u, 0x4140)));
          mma16816<M>(acc[4 * y + 1], pf, biased_to_half2(__byte_perm(a01, 0x64646464u, 0x4342)),
                      biased_to_half2(__byte_perm(c01, 0x64646464u, 0x4342)));
          mma16816<M>(acc[4 * y + 2], pf, biased_to_half2(__byte_perm(a23, 0x64646464u, 0x4140)),
                      biased_to_half2(__byte_perm(c23, 0x64646464u, 0x4140)));
          mma16816<M>(acc[4 * y + 3], pf, biased_to_half2(__byte_perm(a23, 0x64646464u, 0x4342)),
                      biased_to_half2(__byte_perm(c23, 0x64646464u, 0x4342)));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + s);
    }

    // ---- join the four warps
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t == 0) {
        float* x = ml + (warp * kDecRows + g + 8 * r) * 4;
        x[0] = m1[r];
        x[1] = l[r];
        x[2] = I8 ? m2[r] : m1[r];
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kDecWarps * 32) : "memory");
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mo = -INFINITY;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) mo = fmaxf(mo, ml[(w * kDecRows + g + 8 * r) * 4 + 2]);
      const float f = ex2_approx((I8 ? m2[r] : m1[r]) - (mo == -INFINITY ? 0.0f : mo));
      float* dst = red + (warp * kDecRows + g + 8 * r) * C::RED_STRIDE;
      if constexpr (!I8) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
          *reinterpret_cast<float2*>(dst + x * 8 + 2 * t) = make_float2(acc[x][2 * r] * f, acc[x][2 * r + 1] * f);
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int x = 0; x < NT; x += 4)
            *reinterpret_cast<float4*>(dst + (2 * t + c) * (D / 8) + x) =
                make_float4(acc[x][2 * r + c] * f, acc[x + 1][2 * r + c] * f, acc[x + 2][2 * r + c] * f,
                            acc[x + 3][2 * r + c] * f);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kDecWarps * 32) : "memory");
    const bool begins = t0 == 0, ends = t0 + n == ts.count;
    const int slot = 2 * cta + (begins ? 1 : 0);
#pragma unroll
    for (int x = 0; x < kDecRows * (D / 4) / (kDecWarps * 32); ++x) {
      const int idx = x * kDecWarps * 32 + threadIdx.x;
      const int row = idx / (D / 4), c4 = idx % (D / 4);
      if (row >= rows) continue;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float ms = -INFINITY, mo = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(red + (w * kDecRows + row) * C::RED_STRIDE + c4 * 4);
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
        ms = fmaxf(ms, ml[(w * kDecRows + row) * 4]);
        mo = fmaxf(mo, ml[(w * kDecRows + row) * 4 + 2]);
      }
      const float use = ms == -INFINITY ? 0.0f : ms;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        const float* y = ml + (w * kDecRows + row) * 4;
        sum = fmaf(y[1], ex2_approx(y[0] - use), sum);
      }
      if (begins && ends) {
        // INT8: the output is relative to the maximum of the weights, the sum to that of the scores
        const float inv = sum == 0.0f ? 0.0f : (I8 ? ex2_approx(mo - use) / sum : 1.0f / sum);
        const int fr = mt * kDecRows + row, tok = fr / p.G, hd = fr - tok * p.G;
        T* dst = static_cast<T*>(p.o) + (int64_t)(sq.base + tok) * p.o_st + (int64_t)(h * p.G + hd) * p.o_sh + c4 * 4;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
      } else {
        *reinterpret_cast<float4*>(p.part + ((int64_t)slot * kDecRows + row) * D + c4 * 4) = o;
        if (c4 == 0) *reinterpret_cast<float4*>(p.part_ml + (slot * kDecRows + row) * 4) = make_float4(ms, sum, mo, 0.0f);
      }
    }
    if (begins && !ends) cut = make_int4(b, h, mt, (int)((ts.count - n + per - 1) / per));
    asm volatile("bar.sync 1, %0;" ::"n"(kDecWarps * 32) : "memory");
    rem += n;
    left -= n;
  }
  if (threadIdx.x == 0) p.desc[cta] = cut;
}

// Joins the pieces of items that the pieces' borders cut: the item that piece c begins without ending
// (slot 2 c + 1) has its other parts in slots 2 c' of the pieces that follow. Block (c, row) joins one
// row: eight warps share its parts, lanes hold D / 32 channels each.
constexpr int kCombineThreads = 256;
template <int D, bool I8, typename T>
__global__ void __launch_bounds__(kCombineThreads) paged_combine_kernel(const DecodeParams p) {
  constexpr int E = D / 32, W = kCombineThreads / 32;
  __shared__ float s_o[W][D];
  __shared__ float s_ml[W][3];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 d = p.desc[blockIdx.x];
  if (d.w == 0) return;
  const int warp = warp_id(), lane = lane_id(), row = blockIdx.y;
  const PagedSeq sq = paged_seq(p.s, d.x);
  const int fr = d.z * kDecRows + row;
  if (fr >= sq.n * p.G) return;
  const int tok = fr / p.G, hd = fr - tok * p.G;
  float o[E], ms = -INFINITY, l = 0.0f, mo = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll 4
  for (int j = warp; j <= d.w; j += W) {
    const int64_t slot = j == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + j);
    const float4 x = *reinterpret_cast<const float4*>(p.part_ml + (slot * kDecRows + row) * 4);
    const float* src = p.part + (slot * kDecRows + row) * D + lane * E;
    float v[E];
    if constexpr (E == 4) {
      const float4 y = *reinterpret_cast<const float4*>(src);
      v[0] = y.x; v[1] = y.y; v[2] = y.z; v[3] = y.w;
    } else {
      const float2 y = *reinterpret_cast<const float2*>(src);
      v[0] = y.x; v[1] = y.y;
    }
    const float mn = fmaxf(ms, x.x), us = mn == -INFINITY ? 0.0f : mn;
    l = fmaf(l, ex2_approx(ms - us), x.y * ex2_approx(x.x - us));
    ms = mn;
    const float on = fmaxf(mo, x.z), uo = on == -INFINITY ? 0.0f : on;
    const float fa = ex2_approx(mo - uo), fb = ex2_approx(x.z - uo);
    mo = on;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], fa, v[e] * fb);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
  if (lane == 0) {
    s_ml[warp][0] = ms;
    s_ml[warp][1] = l;
    s_ml[warp][2] = mo;
  }
  __syncthreads();
  if (warp != 0) return;
  ms = mo = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    ms = fmaxf(ms, s_ml[w][0]);
    mo = fmaxf(mo, s_ml[w][2]);
  }
  l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
  const float us = ms == -INFINITY ? 0.0f : ms, uo = mo == -INFINITY ? 0.0f : mo;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    l = fmaf(s_ml[w][1], ex2_approx(s_ml[w][0] - us), l);
    const float f = ex2_approx(s_ml[w][2] - uo);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(s_o[w][lane * E + e], f, o[e]);
  }
  const float inv = l == 0.0f ? 0.0f : (I8 ? ex2_approx(mo - us) / l : 1.0f / l);
  T* dst = static_cast<T*>(p.o) + (int64_t)(sq.base + tok) * p.o_st + (int64_t)(d.y * p.G + hd) * p.o_sh + lane * E;
  if constexpr (E == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack2<T>(o[0] * inv, o[1] * inv);
}

}  // namespace sage
