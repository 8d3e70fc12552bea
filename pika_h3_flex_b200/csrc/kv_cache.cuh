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

// n / d for 0 <= n < 2^31 by one multiplication: m = ceil(2^(31 + s) / d), 2^(s - 1) < d <= 2^s
struct FastDiv {
  uint32_t m;
  int shift;  // 31 + s
  __host__ static FastDiv of(uint32_t d) {
    int s = 0;
    while ((1ull << s) < d) ++s;
    return FastDiv{static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d), 31 + s};
  }
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * m) >> shift);
  }
};

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
  FastDiv by_page;                                            // division by page_size
  int rows;                                                   // rows of the packed tensors
  int* status;
};

__device__ __forceinline__ void report_cache(const CacheArgs& a, int b) {
  if (a.status) atomicCAS(a.status, 0, kBadCacheIndex | ((b & 0x7FFFFF) << 8));
}

// Whether an earlier launch, or an earlier block of this one, has set the status word: one verdict for the whole block, whose
// threads go on to share memory.
__device__ __forceinline__ bool block_stops(const CacheArgs& a) {
  if (a.status == nullptr) return false;
  return __syncthreads_or(*reinterpret_cast<volatile int*>(a.status) != 0) != 0;
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

// Where a row lives: its sequence's page and the place in it.
struct RowPlace {
  int id, at;
  int state;  // 0: not a row of any sequence (leave everything alone); 1: no position in the cache, or refused; 2: fine
};
__device__ __forceinline__ RowPlace place_of_row(const CacheArgs& a, int t) {
  RowPlace p{0, 0, 0};
  const int b = sequence_of_row(a, t);
  if (b < 0) return p;
  p.state = 1;
  const CacheSeq q = cache_seq(a, b);
  const int pos = q.len - q.n + (t - q.s0);
  if (pos < 0) return p;
  const int slot = a.by_page(pos);
  p.at = pos - slot * a.page_size;
  p.id = __ldg(a.pages + b * a.pages_stride + slot);
  if (static_cast<unsigned>(p.id) >= static_cast<unsigned>(a.n_pages)) {
    report_cache(a, b);
    return p;
  }
  p.state = 2;
  return p;
}

constexpr int kRowThreads = 256;
constexpr int kRowGroups = kRowThreads / 16;  // half-warps of a block

// the larger magnitude of each half, its sign arbitrary; NaN wins
__device__ __forceinline__ uint32_t max_abs_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// A half-warp moves rows of 128 values, 16 lanes x 8 values each: all heads of K and V of one token, or, when there are few
// tokens, a part of them (per_token half-warps and gridDim.y blocks share a token).  The token's place is looked up once;
// inside the loop an address is an addition away.  K and V rows of kUnroll heads are in flight per half-warp.
// Quantising is bound by instructions rather than by memory: looking every (token, head) row up by itself, with a division
// and a search each, took 688 us (clip of 49,384 x 40 heads into e4m3), computing every address by multiplication, with what
// rows of NaN need in every row's way, 333 us; now it takes 277 us, 5.5 TB/s.  Reading it back takes 249 us, 6.1 TB/s;
// unquantised 325 us in and 313 us out, 6.2 and 6.5 TB/s.
// kWrite: packed -> cache; otherwise cache -> packed.
template <bool kWrite, bool kQuantised>
constexpr int kUnroll = kWrite && kQuantised ? 2 : 4;  // quantising wants registers for more warps
// Blocks per SM.  More warps hide the conversions of the quantised forms (write 277 us with 4, 286 with 3; read 249 and 268);
// the plain copies want their registers instead (bf16 write 325 us with 2, 354 with 4; read 313 and 333).
template <bool kQuantised>
constexpr int kRowBlocksPerSm = kQuantised ? 4 : 2;
constexpr int kExpHeads = 128;  // heads of a token between two meetings of the exponent bytes
template <bool kWrite, bool kQuantised>
__global__ void __launch_bounds__(kRowThreads, kRowBlocksPerSm<kQuantised>) cache_rows_kernel(const __grid_constant__ RowsArgs a, const int per_token) {
  if (block_stops(a.c)) return;
  // A row looks at one sequence's numbers; what is wrong with the others' (offsets that decrease, say) shows only here.
  if (a.c.status != nullptr && blockIdx.x == 0 && blockIdx.y == 0)
    for (int b = threadIdx.x; b < a.c.n_seqs; b += kRowThreads) cache_seq(a.c, b);
  constexpr int kHeads = kUnroll<kWrite, kQuantised>, kRows = 2 * kHeads;  // row i: K (i even) or V of head i / 2
  const int lane = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const uint32_t half_mask = (threadIdx.x & 16) ? 0xFFFF0000u : 0x0000FFFFu;
  const int t = blockIdx.x * (kRowGroups / per_token) + grp / per_token;
  RowPlace p{0, 0, 0};
  if (t < a.c.rows) p = place_of_row(a.c, t);
  const int step = per_token * gridDim.y, first_y = grp % per_token + per_token * blockIdx.y;
  // Exponent bytes of a write meet in shared memory, so that the 16 tokens' bytes of a head leave in one store (they are
  // neighbours in memory): a store per byte cost a fifth of the time.  With few tokens each lane stores its own.
  const bool meet = kWrite && kQuantised && step == 1;
  __shared__ uint8_t exp_s[kWrite && kQuantised ? 2 * kExpHeads : 1][kRowGroups];
  __shared__ uint8_t* exp_at[2][kRowGroups];
  if (meet) {
    if (lane < 2) exp_at[lane][grp] = p.state == 2 ? a.c.exps[lane] + p.id * a.c.exp_page[lane] + p.at * a.c.exp_token[lane] : nullptr;
  } else if (p.state == 0 || (kWrite && p.state == 1)) {
    return;
  }
  const bool moves = p.state == 2 || (!kWrite && p.state == 1);
  for (int c0 = 0; c0 < a.c.kv_heads; c0 += kExpHeads) {
    const int c1 = min(a.c.kv_heads, c0 + kExpHeads);
    const int y_first = c0 + first_y;
    long long cache_step[2], packed_step[2], exp_step[2];
    uint8_t *cached[2], *packed[2], *exps[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      cache_step[x] = step * a.c.head_bytes[x];
      packed_step[x] = step * a.head_bytes[x];
      exp_step[x] = step * a.c.exp_head[x];
      cached[x] = a.c.pool[x] + p.id * a.c.page_bytes[x] + p.at * a.c.token_bytes[x] + y_first * a.c.head_bytes[x] + lane * (kQuantised ? 8 : 16);
      packed[x] = a.x[x] + t * a.row_bytes[x] + y_first * a.head_bytes[x] + lane * 16;
      exps[x] = kQuantised ? a.c.exps[x] + p.id * a.c.exp_page[x] + p.at * a.c.exp_token[x] + y_first * a.c.exp_head[x] : nullptr;
    }
#pragma unroll 1
    for (int y0 = y_first; moves && y0 < c1; y0 += step * kHeads) {
      uint4 r[kRows];
      uint32_t e[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        r[i] = make_uint4(0, 0, 0, 0);
        e[i] = 127;
        const int x = i & 1;
        const bool here = y0 + (i >> 1) * step < c1 && p.state == 2;
        if constexpr (kWrite) {
          if (here) r[i] = ldg_stream(packed[x]);
          packed[x] += packed_step[x];
        } else {
          if (here) {
            if constexpr (kQuantised) {
              const uint2 w = __ldg(reinterpret_cast<const uint2*>(cached[x]));
              r[i].x = w.x;
              r[i].y = w.y;
              e[i] = __ldg(exps[x]);
            } else {
              r[i] = ldg_stream(cached[x]);
            }
          }
          cached[x] += cache_step[x];
          if constexpr (kQuantised) exps[x] += exp_step[x];
        }
      }
      if constexpr (kWrite && kQuantised) {
        // the largest magnitude, two rows in the halves of one word
#pragma unroll
        for (int i = 0; i < kRows; i += 2) {
          const uint32_t m0 = max_abs_bf16x2(max_abs_bf16x2(r[i].x, r[i].y), max_abs_bf16x2(r[i].z, r[i].w));
          const uint32_t m1 = max_abs_bf16x2(max_abs_bf16x2(r[i + 1].x, r[i + 1].y), max_abs_bf16x2(r[i + 1].z, r[i + 1].w));
          uint32_t both = max_abs_bf16x2(__byte_perm(m0, m1, 0x5410), __byte_perm(m0, m1, 0x7632));
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) both = max_abs_bf16x2(both, __shfl_xor_sync(half_mask, both, o));
          e[i] = row_exponent(both & 0x7FFFu);
          e[i + 1] = row_exponent((both >> 16) & 0x7FFFu);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int x = i & 1, y = y0 + (i >> 1) * step;
        if (y >= c1) break;  // the same for the whole half-warp
        if constexpr (!kWrite) {
          if constexpr (kQuantised) {
            const uint32_t f = e4m3_factor(e[i]) * 0x10001u, w0 = r[i].x, w1 = r[i].y;
            r[i].x = mul_bf16x2(e4m3_pattern(__byte_perm(w0, 0, 0x1404)), f);
            r[i].y = mul_bf16x2(e4m3_pattern(__byte_perm(w0, 0, 0x3424)), f);
            r[i].z = mul_bf16x2(e4m3_pattern(__byte_perm(w1, 0, 0x1404)), f);
            r[i].w = mul_bf16x2(e4m3_pattern(__byte_perm(w1, 0, 0x3424)), f);
            if (e[i] > kOneStepExp) {
              const uint32_t f2 = e4m3_factor2(e[i]) * 0x10001u;
              r[i] = make_uint4(mul_bf16x2(r[i].x, f2), mul_bf16x2(r[i].y, f2), mul_bf16x2(r[i].z, f2), mul_bf16x2(r[i].w, f2));
            }
          }
          *reinterpret_cast<uint4*>(packed[x]) = r[i];
          packed[x] += packed_step[x];
        } else {
          if constexpr (kQuantised) {
            // 2^-k, exact in bf16 (what it takes below the type's smallest number is a zero in e4m3 anyway)
            const uint32_t f = (254u - min(e[i], 247u)) * 0x800080u;
            const uint32_t w[4] = {mul_bf16x2(r[i].x, f), mul_bf16x2(r[i].y, f), mul_bf16x2(r[i].z, f), mul_bf16x2(r[i].w, f)};
            uint32_t c[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) c[z] = cvt_e4m3x2(__uint_as_float(w[z] << 16), __uint_as_float(w[z] & 0xFFFF0000u));
            if (e[i] >= 247u) {  // rare
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                // the top of the range: a code of 256 would stand for 2^128, 240 is the last one that does not
                const float lo = fminf(fmaxf(__uint_as_float(w[z] << 16), -240.f), 240.f), hi = fminf(fmaxf(__uint_as_float(w[z] & 0xFFFF0000u), -240.f), 240.f);
                c[z] = e[i] == 255u ? 0u : cvt_e4m3x2(lo, hi);  // a row that is not finite has no codes, only its byte
              }
            }
            *reinterpret_cast<uint2*>(cached[x]) = make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
            if (lane == 0) {
              if (meet) exp_s[x * kExpHeads + y - c0][grp] = static_cast<uint8_t>(e[i]);
              else *exps[x] = static_cast<uint8_t>(e[i]);
            }
            exps[x] += exp_step[x];
          } else {
            *reinterpret_cast<uint4*>(cached[x]) = r[i];
          }
          cached[x] += cache_step[x];
        }
      }
    }
    if (meet) {
      __syncthreads();
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint8_t* to = exp_at[x][lane];  // lane: token of the block
        if (to != nullptr)
          for (int y = c0 + grp; y < c1; y += kRowGroups) to[y * a.c.exp_head[x]] = exp_s[x * kExpHeads + y - c0][lane];
      }
      __syncthreads();
    }
  }
}

}  // namespace h3a
