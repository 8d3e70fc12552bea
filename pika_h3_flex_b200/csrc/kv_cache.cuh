// Paged K/V cache: page addressing, and the two kernels that move rows into and out of it.
//
// A cache holds, per K/V head, one row of 128 values per token: bf16, or e4m3 codes with one exponent byte per row.  Row i
// of the n_b new rows of sequence b is the token at position lengths[b] - n_b + i, in page pages[b][position / page_size].
//
// The quantised form divides a row by the smallest power of two 2^k that brings its largest magnitude to at most 448 and
// rounds to e4m3 (nearest even); the byte holds k + 127.  A power of two costs a floating-point code no relative
// precision (absmax / 448 would only use one more bit of the RANGE, 2^-9 .. 2^8.8, of which a row of activations needs
// little), and code * 2^k has 4 significant bits: a bf16 number.  So what is read back, and what the attention multiplies,
// is exactly what is stored.  A row that holds a NaN or an infinity has no such k: byte 255 marks it, and it reads back as
// 128 NaNs.
//
// Both kernels are HBM-bound: 256 B of bf16 and 129 B (256 B unquantised) of cache per row, each moved once.
#pragma once
#include "ptx.cuh"

namespace h3a {

constexpr int kCacheDim = 128;
constexpr int kBadCacheIndex = 10;  // status code: a page, a length or a row offset is outside its range (H3A_ERR_INDEX)

struct CacheArgs {
  uint8_t* pool[2];                                           // K, V
  long long page_bytes[2], token_bytes[2], head_bytes[2];     // strides in bytes
  uint8_t* exps[2];                                           // quantised: exponent bytes
  long long exp_page[2], exp_token[2], exp_head[2];
  const int* pages;
  long long pages_stride;
  const int* lengths;
  const int* starts;
  int n_seqs, max_pages, n_pages, page_size, kv_heads;
  int rows;                                                   // rows of the packed tensors
  int* status;
};

__device__ __forceinline__ void report_cache(const CacheArgs& a, int b) {
  if (a.status) atomicCAS(a.status, 0, kBadCacheIndex | ((b & 0x7FFFFF) << 8));
}

// One sequence of the batch, with every number brought into its range (what is outside is reported).
struct CacheSeq {
  int s0, n, len;
};
__device__ __forceinline__ CacheSeq cache_seq(const CacheArgs& a, int b) {
  const int s0 = __ldg(a.starts + b), s1 = __ldg(a.starts + b + 1), len = __ldg(a.lengths + b);
  CacheSeq q;
  q.s0 = max(0, min(s0, a.rows));
  q.n = max(q.s0, min(s1, a.rows)) - q.s0;
  q.len = max(0, min(len, a.max_pages * a.page_size));
  if (q.s0 != s0 || q.n != s1 - s0 || q.len != len) report_cache(a, b);
  return q;
}

// 16 bytes that are read once: not worth a line of L1
__device__ __forceinline__ uint4 ldg_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// ---- e4m3 rows
// Two e4m3 codes sit in the HIGH bytes of h's two halves (the low bytes are ignored).  Moved down by four bits, a code's
// exponent and mantissa fields land in a bf16's, whose bias is 120 larger: the pattern is code * 2^-120, e4m3
// subnormals included, and one bf16 multiplication by 2^(120 + k) finishes the job.
__device__ __forceinline__ uint32_t e4m3_pattern(uint32_t h) {
  return ((h & 0x7F007F00u) >> 4) | (h & 0x80008000u);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 2^(120 + k) as bf16 bits for an exponent byte e = k + 127.  Above e = 134 that exceeds the type: the product is then
// taken in two steps, 2^127 first and e4m3_factor2(e) after it.  Byte 255: NaN.
__device__ __forceinline__ uint32_t e4m3_factor(uint32_t e) {
  return e == 255u ? 0x7FFFu : min(e + 120u, 254u) << 7;
}
__device__ __forceinline__ uint32_t e4m3_factor2(uint32_t e) {
  return (e > 134u && e != 255u ? e - 7u : 127u) << 7;
}
constexpr uint32_t kOneStepExp = 134;

// exponent byte of a row whose largest magnitude has the bf16 bits `top` (sign removed)
__device__ __forceinline__ uint32_t row_exponent(uint32_t top) {
  if (top >= 0x7F80u) return 255u;
  const int e = static_cast<int>(top >> 7) - 8 + ((top & 0x7Fu) > 0x60u ? 1 : 0);  // 448 = 1.75 * 2^8; 0x60 = .75 * 128
  return static_cast<uint32_t>(max(e, 7));
}
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

struct RowsArgs {
  CacheArgs c;
  uint8_t* x[2];                        // packed rows, bf16: K, V
  long long row_bytes[2], head_bytes[2];
};

// Sequence that row t belongs to, or -1: the last b with starts[b] <= t, if the row lies inside it.
__device__ __forceinline__ int sequence_of_row(const CacheArgs& a, int t) {
  int lo = 0, hi = a.n_seqs;  // starts[lo] <= t < starts[hi], if there is such a pair
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.starts + mid) <= t) lo = mid;
    else hi = mid;
  }
  return (__ldg(a.starts + lo) <= t && t < __ldg(a.starts + lo + 1)) ? lo : -1;
}

// Where one (row, K or V, head) unit lives: offset of its cached row and of its exponent byte.
struct RowPlace {
  long long cached, exp;
  int state;  // 0: not a row of any sequence, or refused (leave everything alone); 1: no position in the cache; 2: fine
};
__device__ __forceinline__ RowPlace place_of_row(const CacheArgs& a, int t, int x, int h) {
  RowPlace p;
  p.cached = p.exp = 0;
  p.state = 0;
  const int b = sequence_of_row(a, t);
  if (b < 0) return p;
  const CacheSeq q = cache_seq(a, b);
  const int pos = q.len - q.n + (t - q.s0);
  if (pos < 0) {
    p.state = 1;
    return p;
  }
  const int slot = pos / a.page_size, at = pos - slot * a.page_size;
  const int id = __ldg(a.pages + b * a.pages_stride + slot);
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.n_pages)) {
    report_cache(a, b);
    p.state = 1;
    return p;
  }
  p.cached = id * a.page_bytes[x] + at * a.token_bytes[x] + h * a.head_bytes[x];
  p.exp = id * a.exp_page[x] + at * a.exp_token[x] + h * a.exp_head[x];
  p.state = 2;
  return p;
}

constexpr int kRowThreads = 256;
constexpr int kRowUnroll = 4;  // units a half-warp has in flight: 4 x 256 B

// A half-warp owns one row (16 lanes x 16 B) of one head of K or V; consecutive half-warps take consecutive heads, which
// lie next to each other in the packed rows.  kWrite: packed -> cache; otherwise cache -> packed.
template <bool kWrite, bool kQuantised>
__global__ void __launch_bounds__(kRowThreads) cache_rows_kernel(const RowsArgs a) {
  if (a.c.status && *reinterpret_cast<volatile int*>(a.c.status) != 0) return;
  const int lane = threadIdx.x & 15;
  const uint32_t half_mask = (threadIdx.x & 16) ? 0xFFFF0000u : 0x0000FFFFu;
  const uint32_t per_row = 2u * a.c.kv_heads;
  const uint32_t n_units = a.c.rows * per_row;  // below 2^31: checked by the host
  const uint32_t step = gridDim.x * (kRowThreads / 16);
  for (uint32_t u0 = blockIdx.x * (kRowThreads / 16) + (threadIdx.x >> 4); u0 < n_units; u0 += step * kRowUnroll) {
    RowPlace p[kRowUnroll];
    uint4 r[kRowUnroll];
    uint32_t e[kRowUnroll];
    uint8_t* packed[kRowUnroll];
    int x[kRowUnroll];
#pragma unroll
    for (int i = 0; i < kRowUnroll; ++i) {
      const uint32_t u = u0 + i * step;
      p[i].state = 0;
      x[i] = 0;
      e[i] = 0;
      r[i] = make_uint4(0, 0, 0, 0);
      packed[i] = nullptr;
      if (u < n_units) {
        const int t = static_cast<int>(u / per_row);
        const int y = static_cast<int>(u - t * per_row);
        x[i] = y >= a.c.kv_heads;
        const int h = y - x[i] * a.c.kv_heads;
        p[i] = place_of_row(a.c, t, x[i], h);
        packed[i] = a.x[x[i]] + t * a.row_bytes[x[i]] + h * a.head_bytes[x[i]] + lane * 16;
        if (p[i].state == 2) {
          if constexpr (kWrite) {
            r[i] = ldg_stream(packed[i]);
          } else if constexpr (kQuantised) {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(a.c.pool[x[i]] + p[i].cached + lane * 8));
            r[i].x = w.x;
            r[i].y = w.y;
            e[i] = __ldg(a.c.exps[x[i]] + p[i].exp);
          } else {
            r[i] = ldg_stream(a.c.pool[x[i]] + p[i].cached + lane * 16);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kRowUnroll; ++i) {
      if constexpr (kWrite) {
        if constexpr (kQuantised) {
          // the largest magnitude by its bits: finite values order as integers, NaN and infinity lie above them
          uint32_t m = __vmaxu2(__vmaxu2(r[i].x & 0x7FFF7FFFu, r[i].y & 0x7FFF7FFFu), __vmaxu2(r[i].z & 0x7FFF7FFFu, r[i].w & 0x7FFF7FFFu));
          m = max(m >> 16, m & 0xFFFFu);
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(half_mask, m, o));
          const uint32_t ex = row_exponent(m);
          // 2^-k; at the top of the type's range a code of 256 would stand for 2^128: 240 is the last one that does not
          const float f = __uint_as_float((254u - min(ex, 247u)) << 23);
          const float cap = ex == 247u ? 240.0f : 448.0f;
          const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
          uint32_t c[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float lo = __uint_as_float(w[y] << 16) * f, hi = __uint_as_float(w[y] & 0xFFFF0000u) * f;
            c[y] = cvt_e4m3x2(fminf(fmaxf(lo, -cap), cap), fminf(fmaxf(hi, -cap), cap));
          }
          if (p[i].state == 2) {
            *reinterpret_cast<uint2*>(a.c.pool[x[i]] + p[i].cached + lane * 8) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
            if (lane == 0) a.c.exps[x[i]][p[i].exp] = static_cast<uint8_t>(ex);
          }
        } else if (p[i].state == 2) {
          *reinterpret_cast<uint4*>(a.c.pool[x[i]] + p[i].cached + lane * 16) = r[i];
        }
      } else if (p[i].state != 0) {  // a row without a position is zeros (r is)
        if (kQuantised && p[i].state == 2) {
          const uint32_t f = e4m3_factor(e[i]) * 0x10001u, f2 = e4m3_factor2(e[i]) * 0x10001u;
          const uint32_t w0 = r[i].x, w1 = r[i].y;
          r[i].x = mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(w0, 0, 0x1404)), f), f2);
          r[i].y = mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(w0, 0, 0x3424)), f), f2);
          r[i].z = mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(w1, 0, 0x1404)), f), f2);
          r[i].w = mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(w1, 0, 0x3424)), f), f2);
        }
        *reinterpret_cast<uint4*>(packed[i]) = r[i];
      }
    }
  }
}

}  // namespace h3a
