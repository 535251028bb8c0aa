// sage_paged.cuh — the paged key/value cache: where a token lives, and the kernels that write new
// tokens into it and read tokens back.
//
// Token i (of n) newest ones of sequence b, which holds L tokens after them, has position
// p = L - n + i; it lives in page table[b][p / P], row p % P, P a power of two. 16-bit storage
// keeps the values. INT8 storage keeps, per (token, head) row x of D values (K: x - mean of its
// head and channel, where the cache has a mean):
//   a = max |x|, scale = a / 127, code = rint(127 x / a) (ties to even; a = 0: code 0)
// and reads back code * scale (+ mean), rounded once to 16 bits. 127 x is exact in fp32 for 16-bit
// x, and one correctly rounded division follows, so the code is the mathematically nearest one:
// a quotient of integers of <= 18 and <= 11 bits that is no tie is >= 2^-12 away from one, far more
// than half an ulp of a value below 128 (2^-18). A row that holds an infinity or a NaN gets
// a = inf / NaN as its maximum and reads back as NaN.
//
// Both kernels move each byte once (write: 2 D in, 2 D or D + 4 out per row; read the inverse):
// HBM bounds them for prompts, launch latency for single tokens.
//
// Nothing here trusts the device-side arrays: prefix sums are clamped to the packed tensor, lengths
// to the page table's width, and a page number outside the cache is skipped (written) or read as 0.
#pragma once

#include "sage_quant.cuh"
#include "sage_seq.cuh"
#include "sm100_ptx.cuh"

namespace sage {

struct PagedSeqs {
  const int* cu;     // [batch + 1] prefix sums of the new tokens; NULL: one token per sequence
  const int* lens;   // [batch] tokens held, the new ones included
  const int* table;  // [batch][width] page numbers, row stride table_stride
  int64_t table_stride;
  int batch, width;
  int tokens;        // rows of the packed tensor
  int max_new;       // no sequence has more new tokens
  int cap;           // width * page size, clamped to 2^30: no length goes past it
};

struct PagedSeq {
  int base, n, len;  // first packed row, new tokens, tokens held after them
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedSeqs& s, int b) {
  PagedSeq r;
  const int len = s.lens[b];
  if (s.cu == nullptr) {
    r.base = b;
    r.n = b < s.tokens ? 1 : 0;
  } else {
    const SeqSpan sp = seq_span(s.cu, b, s.max_new, s.tokens);
    r.base = sp.base;
    r.n = sp.len;
  }
  r.len = min(max(len, 0), s.cap);
  return r;
}

struct PagedStore {
  void* k;           // [pages][heads][P][D] (any strides): 16-bit values or INT8 codes
  void* v;
  float* k_scale;    // [pages][heads][P]
  float* v_scale;
  const float* k_mean;  // [heads][D], nullable
  int64_t k_sp, k_sh, k_st, v_sp, v_sh, v_st;  // element strides: page, head, token
  int pages, page_shift, heads;
};

struct PagedMoveParams {
  PagedStore c;
  PagedSeqs s;
  void* k;  // packed [tokens][heads][D]
  void* v;
  int64_t k_st, k_sh, v_st, v_sh;
};

// Sequence of packed row `row`: the last b with cu[b] <= row, by 32-ary search of the warp (one
// round of loads per factor of 32 in the batch, two for up to 1024 sequences).
__device__ __forceinline__ int warp_find_seq(const int* cu, int batch, int row) {
  int lo = 0, n = batch;  // the answer is in [lo, lo + n)
  const int lane = threadIdx.x & 31;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool le = at < n && cu[lo + at] <= row;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int hit = max(__popc(m) - 1, 0);
    lo += hit * step;
    n = min(step, n - hit * step);
  }
  return lo;
}

// |x| bits of a float as an integer: ordered like the values, NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

constexpr int kPagedThreads = 256;

// One warp per token: its K and V rows of all heads, 8 values (16 bytes) per lane, D / 8 lanes per
// row. READ = false: write into the cache; true: read out of it. The token's page is looked up
// once for all its 2 * heads rows.
template <int D, typename T, bool I8, bool READ>
__global__ void __launch_bounds__(kPagedThreads) paged_move_kernel(const PagedMoveParams p) {
  constexpr int LPR = D / 8;        // lanes per row
  constexpr int RPW = 32 / LPR;     // rows per warp pass
  constexpr int U = 4;              // passes in flight
  const int lane = threadIdx.x & 31;
  const int64_t token64 = (int64_t)blockIdx.x * (kPagedThreads / 32) + (threadIdx.x >> 5);
  if (token64 >= p.s.tokens) return;
  const int token = (int)token64;
  const int b = p.s.cu ? warp_find_seq(p.s.cu, p.s.batch, token) : token;
  if (b >= p.s.batch) return;
  const PagedSeq sq = paged_seq(p.s, b);
  const int i = token - sq.base;
  if (i < 0 || i >= sq.n) return;  // a row behind the last sequence: left as it is
  const int pos = sq.len - sq.n + i;
  int page = -1;
  if (pos >= 0) page = p.s.table[(int64_t)b * p.s.table_stride + (pos >> p.c.page_shift)];
  const bool in = page >= 0 && page < p.c.pages;
  if (!READ && !in) return;
  const int row = pos & ((1 << p.c.page_shift) - 1);
  const int g = lane % LPR, sub = lane / LPR;
  const int n_rows = 2 * p.c.heads;  // K rows, then V rows
  for (int r0 = 0; r0 < n_rows; r0 += RPW * U) {
    uint4 raw[U];
    float sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * RPW + sub;
      const bool ok = r < n_rows;
      const bool isv = r >= p.c.heads;
      const int h = isv ? r - p.c.heads : r;
      raw[u] = make_uint4(0u, 0u, 0u, 0u);
      sc[u] = 0.0f;
      if constexpr (READ) {
        if (ok && in) {
          const char* base = static_cast<const char*>(isv ? p.c.v : p.c.k);
          const int64_t off = isv ? page * p.c.v_sp + h * p.c.v_sh + row * p.c.v_st
                                  : page * p.c.k_sp + h * p.c.k_sh + row * p.c.k_st;
          if constexpr (I8) {
            const uint2 w = *reinterpret_cast<const uint2*>(base + off + g * 8);
            raw[u].x = w.x;
            raw[u].y = w.y;
            sc[u] = (isv ? p.c.v_scale : p.c.k_scale)[(((int64_t)page * p.c.heads + h) << p.c.page_shift) + row];
          } else {
            raw[u] = *reinterpret_cast<const uint4*>(base + (off + g * 8) * 2);
          }
        }
      } else {
        if (ok) {
          const char* base = static_cast<const char*>(isv ? p.v : p.k);
          const int64_t off = isv ? token * p.v_st + h * p.v_sh : token * p.k_st + h * p.k_sh;
          raw[u] = ldg_nc_v4(base + (off + g * 8) * 2);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * RPW + sub;
      const bool ok = r < n_rows;
      const bool isv = r >= p.c.heads;
      const int h = isv ? r - p.c.heads : r;
      const float* mean = (I8 && ok && !isv && p.c.k_mean) ? p.c.k_mean + h * D + g * 8 : nullptr;
      if constexpr (READ) {
        if (!ok) continue;
        const int64_t off = isv ? token * p.v_st + h * p.v_sh : token * p.k_st + h * p.k_sh;
        uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(isv ? p.v : p.k) + (off + g * 8) * 2);
        if constexpr (I8) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t w = e < 4 ? raw[u].x : raw[u].y;
            f[e] = __fmul_rn((float)(int8_t)(w >> (8 * (e & 3))), sc[u]);
            if (mean && in) f[e] = __fadd_rn(f[e], mean[e]);
          }
          *dst = Half8<T>::from_float(f);
        } else {
          *dst = raw[u];
        }
      } else {
        if constexpr (I8) {
          float f[8];
          Half8<T>::to_float(raw[u], f);
          if (mean) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __fsub_rn(f[e], mean[e]);
          }
          uint32_t m = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) m = max(m, abs_bits(f[e]));
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          const float a = __uint_as_float(m);
          int c[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            // NaN (0 / 0, inf / inf) converts to 0
            c[e] = min(max(__float2int_rn(__fdiv_rn(__fmul_rn(f[e], 127.0f), a)), -127), 127);
          }
          if (ok) {
            const int64_t off = isv ? page * p.c.v_sp + h * p.c.v_sh + row * p.c.v_st
                                    : page * p.c.k_sp + h * p.c.k_sh + row * p.c.k_st;
            *reinterpret_cast<uint2*>(static_cast<char*>(isv ? p.c.v : p.c.k) + off + g * 8) =
                make_uint2(pack4_lo_bytes(c[0], c[1], c[2], c[3]), pack4_lo_bytes(c[4], c[5], c[6], c[7]));
            if (g == 0)
              (isv ? p.c.v_scale : p.c.k_scale)[(((int64_t)page * p.c.heads + h) << p.c.page_shift) + row] =
                  __fdiv_rn(a, 127.0f);
          }
        } else if (ok) {
          const int64_t off = isv ? page * p.c.v_sp + h * p.c.v_sh + row * p.c.v_st
                                  : page * p.c.k_sp + h * p.c.k_sh + row * p.c.k_st;
          *reinterpret_cast<uint4*>(static_cast<char*>(isv ? p.c.v : p.c.k) + (off + g * 8) * 2) = raw[u];
        }
      }
    }
  }
}

}  // namespace sage
