// sage_paged.cuh — the paged key/value cache: where a token lives, and the kernels that write new
// tokens into it and read tokens back.
//
// Token i (of n) newest ones of sequence b, which holds L tokens after them, has position
// p = L - n + i; it lives in page table[b][p / P], row p % P, P a power of two. 16-bit storage
// keeps the values. INT8 storage keeps, per (token, head) row x of D values (K: x - mean of its
// head and channel, where the cache has a mean):
//   a = max |x|, scale = a / 127, code = rint(127 x / a) (ties to even; a = 0: code 0)
// and reads back code * scale (+ mean), rounded once to 16 bits. For 16-bit x without a mean 127 x is
// exact in fp32 and one correctly rounded division follows, so the code is the mathematically nearest
// one: with significands X, A < 2^11 and x = 2^-k X, a = A (k >= 0), 127 x / a misses a tie that it is
// not on by at least 1 / (2 A 2^k) > 2^-12-k, while it is below 2^8-k and so rounded by less than
// 2^-16-k. A row that holds an infinity or a NaN gets a = inf / NaN as its maximum and reads back as NaN.
// Two new tokens of a call that name the same place leave either's values, of an INT8 cache possibly
// one's codes under the other's scale.
//
// Both kernels move each byte once (write: 2 D in, 2 D or D + 4 out per row; read the inverse):
// HBM bounds them for prompts, launch latency for single tokens. Measured (B200, 32768 tokens of 8 heads,
// head_dim 128): 16 bit 47 us (5.7 TB/s), INT8 append 46 us (4.4 TB/s; quantising takes 65 % of the issue
// slots; with means 53 us), gather 44 us (4.6 TB/s; issue slots 56 %).
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
  // Sequences whose query rows per key/value head (new tokens * group) lie outside [rows_lo, rows_hi] are
  // left to another launch: they appear to have no new tokens. rows_hi 0: none is.
  int group, rows_lo, rows_hi;
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
  if (s.rows_hi != 0 && (r.n * s.group < s.rows_lo || r.n * s.group > s.rows_hi)) r.n = 0;
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
  int per_shift;  // log2 of the tokens per block
};

// Sequence of packed row `row`: the last b with cu[b] <= row (a search per lane).
__device__ __forceinline__ int find_seq(const int* cu, int batch, int row) {
  int lo = 0, n = batch;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int half = n / 2;
    if (cu[lo + half] <= row) { lo += half; n -= half; }
    else n = half;
  }
  return lo;
}

// |x| bits of a float as an integer: ordered like the values, NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Eight INT8 codes rint(127 f / a) of f, |f| <= a, with the largest |f| of the row a.
__device__ __forceinline__ uint2 codes_of(float (&f)[8], float a) {
  if (!(a > 7.9e-31f && a < 1.2e30f)) {  // beyond 2^-100 .. 2^100 (rare): brought inside by a power of two
    if (!(a > 0.0f && a < INFINITY)) return make_uint2(0u, 0u);
    const float s = a < 1.0f ? 18446744073709551616.0f : 5.421010862427522e-20f;  // 2^64, 2^-64
    a *= s;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= s;
  }
  // The correctly rounded quotient (quotient_rn), two lanes at a time; adding 1.5 * 2^23 rounds it to an
  // integer, ties to even, whose two's complement byte is the sum's lowest.
  const float r = __frcp_rn(a);
  const float2 r2 = make_float2(r, r), na2 = make_float2(-a, -a);
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 x = fmul2(make_float2(f[e], f[e + 1]), make_float2(127.0f, 127.0f));
    const float2 q = fmul2(x, r2);
    const float2 z = fadd2(ffma2(ffma2(na2, q, x), r2, q), make_float2(12582912.0f, 12582912.0f));
    c[e] = __float_as_uint(z.x);
    c[e + 1] = __float_as_uint(z.y);
  }
  return make_uint2(pack4_lo_bytes(c[0], c[1], c[2], c[3]), pack4_lo_bytes(c[4], c[5], c[6], c[7]));
}

// f += sign * mean, one rounding each (sign 1 or -1).
__device__ __forceinline__ void add_mean(float (&f)[8], const float4* mean, float sign) {
  const float4 a = mean[0], z = mean[1];
  const float m[8] = {a.x, a.y, a.z, a.w, z.x, z.y, z.z, z.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = __fmaf_rn(m[e], sign, f[e]);
}

// 32 bytes in one store (a whole sector of the cache), 16-byte aligned addresses as two.
__device__ __forceinline__ void stg_v8(void* dst, const uint4& a, const uint4& z) {
  if ((reinterpret_cast<uintptr_t>(dst) & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
                 "r"(z.x), "r"(z.y), "r"(z.z), "r"(z.w) : "memory");
  } else {
    reinterpret_cast<uint4*>(dst)[0] = a;
    reinterpret_cast<uint4*>(dst)[1] = z;
  }
}

constexpr int kPagedThreads = 256;

// K (blockIdx.y = 0) or V rows of all heads of 2^per_shift tokens (1 .. 32) per block. Every warp
// resolves all of them, a lane each (sequence, position, page: a chain of four or five loads, paid
// once per block); then the warps share the block's rows, tokens running fastest, so that neighbouring
// rows are neighbours in a page and in its scales. A lane moves eight values, of an INT8 cache sixteen
// (fewer address computations and shuffles per value, which bound it there), U rows in flight.
// READ = false: write into the cache; true: read out of it.
template <int D, typename T, bool I8, bool READ>
__global__ void __launch_bounds__(kPagedThreads) paged_move_kernel(const PagedMoveParams p) {
  constexpr int EPL = I8 ? 16 : 8;  // values per lane
  constexpr int LPR = D / EPL, RPW = 32 / LPR, U = I8 ? 2 : 4;
  constexpr int N16 = EPL / 8;      // 16-byte pieces of a lane's 16-bit values
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool isv = blockIdx.y != 0;
  // ---- this lane's token
  int l_token = -1, l_page = -1, l_row = 0;
  {
    const int64_t tok = ((int64_t)blockIdx.x << p.per_shift) + (lane & ((1 << p.per_shift) - 1));
    const int b = tok >= p.s.tokens ? p.s.batch : p.s.cu ? find_seq(p.s.cu, p.s.batch, (int)tok) : (int)tok;
    if (b < p.s.batch) {
      const PagedSeq sq = paged_seq(p.s, b);
      const int i = (int)tok - sq.base;
      if (i >= 0 && i < sq.n) {  // else a row behind the last sequence: left as it is
        l_token = (int)tok;
        const int pos = sq.len - sq.n + i;
        if (pos >= 0) l_page = p.s.table[(int64_t)b * p.s.table_stride + (pos >> p.c.page_shift)];
        l_row = pos & ((1 << p.c.page_shift) - 1);
        if (l_page < 0 || l_page >= p.c.pages) l_page = -1;
        if (!READ && l_page < 0) l_token = -1;  // nowhere to write
      }
    }
  }
  // strides in 16-byte units, below 2^31: one widening multiply each
  const uint32_t c_sp = (uint32_t)((isv ? p.c.v_sp : p.c.k_sp) >> (I8 ? 4 : 3));
  const uint32_t c_sh = (uint32_t)((isv ? p.c.v_sh : p.c.k_sh) >> (I8 ? 4 : 3));
  const uint32_t c_st = (uint32_t)((isv ? p.c.v_st : p.c.k_st) >> (I8 ? 4 : 3));
  const uint32_t x_st = (uint32_t)((isv ? p.v_st : p.k_st) >> 3), x_sh = (uint32_t)((isv ? p.v_sh : p.k_sh) >> 3);
  const int g = lane % LPR, sub = lane / LPR;
  char* cache = static_cast<char*>(isv ? p.c.v : p.c.k) + g * 16;
  char* packed = static_cast<char*>(isv ? p.v : p.k) + g * (16 * N16);
  float* scales = isv ? p.c.v_scale : p.c.k_scale;
  const float* means = isv || !I8 ? nullptr : p.c.k_mean;
  const int n_rows = p.c.heads << p.per_shift;
  for (int r0 = warp * RPW * U; r0 < n_rows; r0 += (kPagedThreads / 32) * RPW * U) {
    uint4 raw[U][N16];
    float sc[U];
    char *at_cache[U], *at_packed[U];
    int64_t at_scale[U];
    int token[U], page[U], head[U];  // token -1: nothing to do
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * RPW + sub, slot = r & ((1 << p.per_shift) - 1);
      token[u] = __shfl_sync(0xffffffffu, l_token, slot);
      page[u] = __shfl_sync(0xffffffffu, l_page, slot);
      const int row = __shfl_sync(0xffffffffu, l_row, slot);
      head[u] = r >> p.per_shift;
      if (r >= n_rows) token[u] = -1;
      at_cache[u] = cache + (((uint64_t)(uint32_t)page[u] * c_sp + (uint64_t)(uint32_t)head[u] * c_sh + (uint64_t)(uint32_t)row * c_st) << 4);
      at_packed[u] = packed + (((uint64_t)(uint32_t)token[u] * x_st + (uint64_t)(uint32_t)head[u] * x_sh) << 4);
      at_scale[u] = (((int64_t)page[u] * p.c.heads + head[u]) << p.c.page_shift) + row;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      sc[u] = 0.0f;
#pragma unroll
      for (int x = 0; x < N16; ++x) raw[u][x] = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (READ) {
        if (token[u] >= 0 && page[u] >= 0) {
          raw[u][0] = ldg_nc_v4(at_cache[u]);
          if constexpr (I8) sc[u] = __ldg(scales + at_scale[u]);
        }
      } else if (token[u] >= 0) {
#pragma unroll
        for (int x = 0; x < N16; ++x) raw[u][x] = ldg_nc_v4(at_packed[u] + 16 * x);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool ok = token[u] >= 0;
      const float4* mean = (ok && means) ? reinterpret_cast<const float4*>(means + head[u] * D + g * EPL) : nullptr;
      if constexpr (!I8) {
        if (ok) *reinterpret_cast<uint4*>(READ ? at_packed[u] : at_cache[u]) = raw[u][0];
      } else if constexpr (READ) {
        if (!ok) continue;
        const uint32_t w[4] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w};
        uint4 out[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            // byte c + 128 under the exponent of 2^23 is the float 2^23 + 128 + c
            const uint32_t v = w[2 * x + e / 4] ^ 0x80808080u;
            const float2 b = make_float2(__uint_as_float(__byte_perm(v, 0x4B000000u, 0x7540 + (e & 3))),
                                         __uint_as_float(__byte_perm(v, 0x4B000000u, 0x7541 + (e & 3))));
            const float2 y = fmul2(fadd2(b, make_float2(-8388736.0f, -8388736.0f)), make_float2(sc[u], sc[u]));
            f[e] = y.x;
            f[e + 1] = y.y;
          }
          if (mean && page[u] >= 0) add_mean(f, mean + 2 * x, 1.0f);
          out[x] = Half8<T>::from_float(f);
        }
        stg_v8(at_packed[u], out[0], out[1]);
      } else {
        float f[2][8];
        float a;  // max |f| of the row, a NaN above all
#pragma unroll
        for (int x = 0; x < 2; ++x) Half8<T>::to_float(raw[u][x], f[x]);
        if (means) {  // uniform
          uint32_t m = 0;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (mean) add_mean(f[x], mean + 2 * x, -1.0f);
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, abs_bits(f[x][e]));
          }
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          a = __uint_as_float(m);
        } else {  // of the 16-bit values, as packed integers: ordered like the magnitudes
          uint32_t m = 0;
#pragma unroll
          for (int x = 0; x < 2; ++x)
            m = __vmaxu2(__vmaxu2(m, __vmaxu2(raw[u][x].x & 0x7fff7fffu, raw[u][x].y & 0x7fff7fffu)),
                         __vmaxu2(raw[u][x].z & 0x7fff7fffu, raw[u][x].w & 0x7fff7fffu));
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
          const float2 two = Half8<T>::pair(__vmaxu2(m, m >> 16));
          a = two.x;
        }
        const uint2 c0 = codes_of(f[0], a), c1 = codes_of(f[1], a);
        if (ok) {
          *reinterpret_cast<uint4*>(at_cache[u]) = make_uint4(c0.x, c0.y, c1.x, c1.y);
          if (g == 0) scales[at_scale[u]] = __fdiv_rn(a, 127.0f);
        }
      }
    }
  }
}

}  // namespace sage
