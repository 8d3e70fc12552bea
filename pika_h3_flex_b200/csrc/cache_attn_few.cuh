// Attention of few new rows over a paged K/V cache: up to 16 query rows per K/V head and item (one token with its group of
// heads, or a few tokens).
//
// HBM-bound: the cache is read once, 2 x 256 B (2 x 129 B) per key and head.  So no shared memory and no tensor-memory
// round trip on the way: a warp takes 16 keys of every tile and loads them straight into the register fragments of the
// warp-level MMA (m16n8k16), with the KEYS (for P V: the dims) as its 16 rows and 8 or 16 query rows as columns: with the
// query rows as the 16 a token with its 5 or 8 heads would leave half of every MMA empty, and the MMAs, not the loads, set
// the pace.  The MMA leaves the order of the contraction free: for K Q^T a lane's 16-byte pieces of a K row ARE its share
// of the k-steps (Q is permuted alike, once per piece); for V^T P^T it loads 16-byte pieces of the four keys its fragment
// needs, paired by byte permutes, and a lane ends up with 16 dims of two rows; P^T turns into an operand through one
// 8 x 8 register transpose per 8 keys.  K of the next 16 keys is requested as soon as K Q^T has consumed this one's
// registers, V after P V.  Blocks are small (4 warps) so that many warps of an SM work on different items.
//
// e4m3: codes become fp16 (exact) in one conversion per pair; the powers of two stay outside the MMA.  A K row's multiplies
// its column of S; Q is scaled to fp16 by a power of two per row that joins the softmax scale.  A V row's multiplies its
// probability, relative to the running reference `vr`, in whose units O is kept.  fp16 holds a product p 2^(v - vr) to
// 2^-31 of the row's largest, far below the rounding of P itself, as long as v - vr stays within 2^-8; a block of keys
// whose exponents lie elsewhere takes bf16 MMAs with the power multiplied into the codes.  The integer route for every
// block (5 instead of 1.5 instructions per pair) ran at 40 % of the HBM rate.
//
// Measured: one token over each of two contexts of 65,537 and 131,072 bf16 keys (40 heads on 8) 127 us, 6.3 TB/s; 64
// contexts of 8,000 keys, 16 heads of their own, bf16 607 to 628 us, 6.7 to 6.9 TB/s, e4m3 361 us, 5.9 TB/s (some 500 instructions per 16
// keys and warp, waiting for memory most of the time; reading two steps ahead into L2, and 3 or 5 blocks per SM instead of
// 4, were not faster); 32 contexts of 200 to 16,384 e4m3 keys 59 us.  Calls of a few microseconds are latency: one token over
// 1,023 bf16 keys takes 12 to 16 us, 3 of them memory's.
#pragma once
#include "cache_attn.cuh"

namespace h3a {

constexpr int kFewRows = 16;     // at most
constexpr int kFewWarps = 4;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewKeyShift = 6;  // 64 keys per tile: 16 per warp
// blocks per SM that the registers allow; kNT: groups of 8 query rows
template <bool kFp8, int kNT>
constexpr int kFewBlocksPerSm = kFp8 && kNT == 1 ? 4 : 3;
constexpr int kFewORow = kCacheDim + 4;        // padded row of O in shared memory

template <int kNT>
struct FewSmem {
  static constexpr int kRows = 8 * kNT;
  float o[kFewWarps][kRows][kFewORow];
  float m[kFewWarps][kRows], l[kFewWarps][kRows];
  alignas(16) uint32_t q[8][32][2 * kNT];   // [k-step][lane] B fragments, bf16
  alignas(16) uint32_t qh[8][32][2 * kNT];  // e4m3: the same in fp16, scaled
  float q_scale[kRows];     // e4m3: 2^(what qh was divided by)
  int poison;               // some V value that only part of the item's rows see is not finite
  // the share's state lives here, not in every thread's registers
  ShareIter iter;
  Piece piece;
  int more;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// transposes an 8 x 8 matrix of 16-bit values held as an MMA fragment
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <bool kFp8, int kNT>
__global__ void __launch_bounds__(kFewThreads, (kFewBlocksPerSm<kFp8, kNT>)) cache_attn_few_kernel(const __grid_constant__ CacheAttnArgs a) {
  extern __shared__ __align__(16) uint8_t few_raw[];
  FewSmem<kNT>& sm = *reinterpret_cast<FewSmem<kNT>*>(few_raw);
  __shared__ ShareStart start;
  if (block_stops(a.c)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  constexpr int kRows = 8 * kNT;
  constexpr int kKW = kFp8 ? 2 : 4;  // 16-byte pieces per lane of a K row
  constexpr int kVW = kFp8 ? 1 : 2;  // ... of a V row

  allow_next_launch();
  {
    ShareIter iter = share_begin(a, &start);
    if (threadIdx.x == 0) {
      a.desc[kDescInts * blockIdx.x] = 0;
      sm.poison = 0;
      sm.more = iter.next(a, sm.piece);
      sm.iter = iter;
    }
  }
  const Piece& p = sm.piece;
  for (;;) {
    __syncthreads();  // the piece is there
    if (!sm.more) return;
    const int r0 = p.it * kRows;
    const int n_rows = min(kRows, p.s.n * a.group - r0);
    const int lim_min = key_limit(a, p.s, a.by_group(r0));
    const int lim_max = key_limit(a, p.s, item_last_token(a, p.s, p.it));

    // O^T: [i][j] holds, of dims (2 j, gid) and (2 j + 1, gid) of the loads' order, rows 8 i + 2 tig + {0, 1}
    float o[kNT][8][4];
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
    float m[kNT][2], l[kNT][2];
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      m[i][0] = m[i][1] = kNoMax;
      l[i][0] = l[i][1] = 0.f;
    }
    uint32_t vr = 0;  // e4m3: O is in units of 2^(vr - 127); 0: none yet

    // The warp's 16 keys of tile t.  Its page number is fetched a step before its rows.
    const int end_key = min(lim_max, p.t1 << kFewKeyShift);
    int key0 = (p.t0 << kFewKeyShift) + warp * 16;
    const int* table = a.c.pages + p.b * a.c.pages_stride;
    uint4 k[2 * kKW], v[4 * kVW];
    uint32_t e = 0;  // lanes 0-15: exponent byte of K row `lane`; lanes 16-31: of V row `lane - 16`
    auto raw_page = [&](int key) { return key < end_key ? __ldg(table + a.c.by_page(key)) : 0; };
    auto check_page = [&](int id) -> int {
      if (static_cast<unsigned>(id) < static_cast<unsigned>(a.c.n_pages)) return id;
      report_cache(a.c, p.b);
      return 0;
    };
    // where this lane's parts of row 0 of page 0 are
    const uint8_t* const k_at = a.c.pool[0] + p.h * a.c.head_bytes[0] + gid * a.c.token_bytes[0] + 16 * tig;
    const uint8_t* const v_at = a.c.pool[1] + p.h * a.c.head_bytes[1] + 2 * tig * a.c.token_bytes[1] + 16 * gid;
    const int ex = lane >> 4;
    const uint8_t* const e_at = kFp8 ? a.c.exps[ex] + p.h * a.c.exp_head[ex] + (lane & 15) * a.c.exp_token[ex] : nullptr;
    auto place = [&](int key) { return key - a.c.by_page(key) * a.c.page_size; };
    auto load_k = [&](int id, int at) {
      const uint8_t* src = k_at + id * a.c.page_bytes[0] + at * a.c.token_bytes[0];
#pragma unroll
      for (int u = 0; u < 2; ++u, src += 8 * a.c.token_bytes[0])
#pragma unroll
        for (int x = 0; x < kKW; ++x) k[u * kKW + x] = ldg_stream(src + 64 * x);
      if constexpr (kFp8) e = __ldg(e_at + id * a.c.exp_page[ex] + at * a.c.exp_token[ex]);
    };
    auto load_v = [&](int id, int at) {
      const uint8_t* src = v_at + id * a.c.page_bytes[1] + at * a.c.token_bytes[1];
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int x = 0; x < kVW; ++x) v[y * kVW + x] = ldg_stream(src + ((y & 1) + 8 * (y >> 1)) * a.c.token_bytes[1] + 128 * x);
    };

    int id = 0, at = 0;
    if (key0 < end_key) {
      id = check_page(raw_page(key0));
      at = place(key0);
      load_k(id, at);
      load_v(id, at);
    }
    // ---- Q as B fragments, dims in the order of the K loads below: half-warps load rows, 8 dims per lane
#pragma unroll
    for (int r = threadIdx.x >> 4; r < kRows; r += kFewThreads / 16) {
      const int l = threadIdx.x & 15;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (r < n_rows) {
        const int token = a.by_group(r0 + r), head = p.h * a.group + (r0 + r) - token * a.group;
        w = __ldg(reinterpret_cast<const uint4*>(a.q + (p.s.s0 + token) * a.q_row_bytes + head * a.q_head_bytes + 16 * l));
      }
      // bf16: piece x = dims 32 x + 8 t + [0, 8) of lane group t; e4m3: pieces 2 c, 2 c + 1 = dims 64 c + 16 t + [0, 16)
      const int x = kFp8 ? 2 * (l >> 3) + (l & 1) : l >> 2, t = kFp8 ? (l & 7) >> 1 : l & 3;
      const int to = (r & 7) * 4 + t, y = r >> 3;
      sm.q[2 * x][to][2 * y] = w.x;
      sm.q[2 * x][to][2 * y + 1] = w.y;
      sm.q[2 * x + 1][to][2 * y] = w.z;
      sm.q[2 * x + 1][to][2 * y + 1] = w.w;
      if constexpr (kFp8) {
        uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync((threadIdx.x & 16) ? 0xFFFF0000u : 0x0000FFFFu, m, o));
        const int e = max(static_cast<int>(max(m >> 16, m & 0xFFFFu) >> 7) - 127 - 4, -120);  // the row's largest: 2^4 .. 2^5
        const float f = pow2_float(-e);
        const uint32_t in[4] = {w.x, w.y, w.z, w.w};
        uint32_t h[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) h[z] = pack_f16x2(__uint_as_float(in[z] << 16) * f, __uint_as_float(in[z] & 0xFFFF0000u) * f);
        sm.qh[2 * x][to][2 * y] = h[0];
        sm.qh[2 * x][to][2 * y + 1] = h[1];
        sm.qh[2 * x + 1][to][2 * y] = h[2];
        sm.qh[2 * x + 1][to][2 * y + 1] = h[3];
        if (l == 0) sm.q_scale[r] = pow2_float(e);
      }
    }
    __syncthreads();
    // this lane's query rows: 8 i + 2 tig + c
    int lim[kNT][2];
    float q_unit[kNT][2];  // e4m3: what the logits of the fp16 fragments are multiplied by
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 8 * i + 2 * tig + c;
        lim[i][c] = r < n_rows ? key_limit(a, p.s, a.by_group(r0 + r)) : 0;
        q_unit[i][c] = kFp8 ? fmaxf(sm.q_scale[r] * a.scale_log2, kLeastUnit) : 0.f;
      }
    int id_next = raw_page(key0 + (1 << kFewKeyShift));
    for (; key0 < end_key; key0 += 1 << kFewKeyShift) {
      const int next = key0 + (1 << kFewKeyShift);
      const bool partly = key0 + 16 > lim_min;  // some row does not see some key (or a row is not there at all)
      // ---- e4m3: exponents of the keys this lane has a row of in S^T, gid and gid + 8: K in byte 0, V in byte 1
      uint32_t ke[2] = {0, 0};
      const uint32_t e_now = e;
      bool fast_k = true, fast_v = true;
      if constexpr (kFp8) {
        const bool gone = key0 + (lane & 15) >= lim_max;
        const uint32_t both = e | (__shfl_down_sync(0xFFFFFFFFu, e, 16) << 8);
        ke[0] = __shfl_sync(0xFFFFFFFFu, both, gid);
        ke[1] = __shfl_sync(0xFFFFFFFFu, both, gid + 8);
        const bool odd = !gone && (lane < 16 ? e > 230u : e > vr || e + 8u < vr);
        if (__any_sync(0xFFFFFFFFu, odd)) {
          fast_k = !__any_sync(0xFFFFFFFFu, lane < 16 && odd);
          const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, lane >= 16 && !gone && e != 255u ? e : 0u);
          if (top > vr) {
            const float f = vr == 0u ? 0.f : pow2_float(static_cast<int>(vr) - static_cast<int>(top));
#pragma unroll
            for (int i = 0; i < kNT; ++i)
#pragma unroll
              for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[i][j][c] *= f;
            vr = top;
          }
          fast_v = !__any_sync(0xFFFFFFFFu, lane >= 16 && !gone && (e > vr || e + 8u < vr));
        }
      }
      // ---- S^T = K Q^T
      float s[kNT][4];
      float unit[kNT][2];
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
        unit[i][0] = unit[i][1] = a.scale_log2;
      }
      if constexpr (!kFp8) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint4 &w0 = k[x >> 1], &w1 = k[kKW + (x >> 1)];
          const uint4 kf = (x & 1) ? make_uint4(w0.z, w1.z, w0.w, w1.w) : make_uint4(w0.x, w1.x, w0.y, w1.y);
#pragma unroll
          for (int i = 0; i < kNT; ++i) mma_bf16(s[i], kf, sm.q[x][lane][2 * i], sm.q[x][lane][2 * i + 1]);
        }
      } else if (fast_k) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t w0 = word_of(k[x >> 2], x & 3), w1 = word_of(k[kKW + (x >> 2)], x & 3);
          const uint4 kf = make_uint4(e4m3_to_f16x2(w0), e4m3_to_f16x2(w1), e4m3_high_to_f16x2(w0), e4m3_high_to_f16x2(w1));
#pragma unroll
          for (int i = 0; i < kNT; ++i) mma_f16(s[i], kf, sm.qh[x][lane][2 * i], sm.qh[x][lane][2 * i + 1]);
        }
        const float f0 = __uint_as_float((ke[0] & 0xFFu) << 23), f1 = __uint_as_float((ke[1] & 0xFFu) << 23);
#pragma unroll
        for (int i = 0; i < kNT; ++i) {
          s[i][0] *= f0;
          s[i][1] *= f0;
          s[i][2] *= f1;
          s[i][3] *= f1;
          unit[i][0] = q_unit[i][0];
          unit[i][1] = q_unit[i][1];
        }
      } else {
        const uint32_t g0 = e4m3_factor(ke[0] & 0xFFu) * 0x10001u, h0 = e4m3_factor2(ke[0] & 0xFFu) * 0x10001u;
        const uint32_t g1 = e4m3_factor(ke[1] & 0xFFu) * 0x10001u, h1 = e4m3_factor2(ke[1] & 0xFFu) * 0x10001u;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t w0 = word_of(k[x >> 2], x & 3), w1 = word_of(k[kKW + (x >> 2)], x & 3);
          const uint4 kf = make_uint4(mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(w0, 0, 0x1404)), g0), h0),
                                      mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(w1, 0, 0x1404)), g1), h1),
                                      mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(w0, 0, 0x3424)), g0), h0),
                                      mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(w1, 0, 0x3424)), g1), h1));
#pragma unroll
          for (int i = 0; i < kNT; ++i) mma_bf16(s[i], kf, sm.q[x][lane][2 * i], sm.q[x][lane][2 * i + 1]);
        }
      }
      // the next 16 keys' K and exponents; their page was asked for a step ago, the page after it is asked for now
      if (next < end_key) {
        id = check_page(id_next);
        at = place(next);
        load_k(id, at);
        id_next = raw_page(next + (1 << kFewKeyShift));
      }
      // ---- softmax: s[i][c] is key gid, s[i][2 + c] key gid + 8, of row 8 i + 2 tig + c
      if (partly) {
#pragma unroll
        for (int i = 0; i < kNT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (key0 + gid + 8 * (c >> 1) >= lim[i][c & 1]) s[i][c] = -INFINITY;
      }
      // The reference moves (and O is rescaled) only when a logit exceeds it by more than 2^8: terms stay far inside the
      // range until then, and until then the lanes that share a row need not meet.
      bool grow = false;
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) grow |= fmaxf(s[i][c], s[i][2 + c]) * unit[i][c] > m[i][c] + 8.f;
      if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
        for (int i = 0; i < kNT; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = fmaxf(s[i][c], s[i][2 + c]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
            const float m_new = fmaxf(m[i][c], top * unit[i][c]);
            const float f = ex2_approx(m[i][c] - m_new);
            m[i][c] = m_new;
            l[i][c] *= f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[i][j][c] *= f;
              o[i][j][2 + c] *= f;
            }
          }
      }
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[i][c] = ex2_approx(__fmul_rn(s[i][c], unit[i][c & 1]) - m[i][c & 1]);  // rounded like the maximum: large ones differ by 0
          l[i][c & 1] += s[i][c];
        }
      // ---- O^T += V^T P^T.  P is 0 where a key is masked, so V must be finite there: rows behind the sequence's last key may
      //      hold anything and count as zeros; a value that some of the item's rows see and others do not counts as zero
      //      if it is not finite, and is put back at the end for the rows that see it.
      //      A bf16 P goes in two parts, the rounded one and what the rounding left, at most 2^-16 of a term lost: the MMAs wait
      //      for memory anyway (64 contexts of 8,000 keys 628 us either way, with 16 query rows 175 against 173), and with one
      //      part the results were half as far off again as their own rounding takes them (2.3e-3 against 1.7e-3 of the
      //      norm).  An fp16 P has 3 bits more and goes in one.  The row sum keeps the unrounded terms.
      if (partly) {
        bool bad = false;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const bool gone = key0 + 2 * tig + (y & 1) + 8 * (y >> 1) >= lim_max;
#pragma unroll
          for (int x = 0; x < kVW; ++x) {
            uint4& w = v[y * kVW + x];
            if (gone) w = make_uint4(0, 0, 0, 0);
            if constexpr (!kFp8) {
              bad |= non_finite2(w.x) || non_finite2(w.y) || non_finite2(w.z) || non_finite2(w.w);
              w = make_uint4(finite_or_zero2(w.x), finite_or_zero2(w.y), finite_or_zero2(w.z), finite_or_zero2(w.w));
            }
          }
        }
        if constexpr (kFp8) bad = lane >= 16 && e_now == 255u && key0 + (lane & 15) < lim_max;
        if (bad) sm.poison = 1;
      }
      if (kFp8 && fast_v) {
        // 2^(6 + v - vr); a key that is gone has P = 0 and any byte at all: its factor has to stay finite
        const float f0 = pow2_float(min(static_cast<int>(ke[0] >> 8) - static_cast<int>(vr), 0) + 6);
        const float f1 = pow2_float(min(static_cast<int>(ke[1] >> 8) - static_cast<int>(vr), 0) + 6);
        uint32_t pf[kNT][2];
#pragma unroll
        for (int i = 0; i < kNT; ++i) {
          pf[i][0] = transpose_8x8(pack_f16x2(s[i][0] * f0, s[i][1] * f0));
          pf[i][1] = transpose_8x8(pack_f16x2(s[i][2] * f1, s[i][3] * f1));
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t x0 = word_of(v[0], w), x1 = word_of(v[kVW], w), x2 = word_of(v[2 * kVW], w), x3 = word_of(v[3 * kVW], w);
          const uint32_t a0 = __byte_perm(x0, x1, 0x5140), a1 = __byte_perm(x0, x1, 0x7362);  // bytes 0, 1 and 2, 3 of both keys
          const uint32_t b0 = __byte_perm(x2, x3, 0x5140), b1 = __byte_perm(x2, x3, 0x7362);
          const uint4 v0 = make_uint4(e4m3_to_f16x2(a0), e4m3_high_to_f16x2(a0), e4m3_to_f16x2(b0), e4m3_high_to_f16x2(b0));
          const uint4 v1 = make_uint4(e4m3_to_f16x2(a1), e4m3_high_to_f16x2(a1), e4m3_to_f16x2(b1), e4m3_high_to_f16x2(b1));
#pragma unroll
          for (int i = 0; i < kNT; ++i) {
            mma_f16(o[i][2 * w], v0, pf[i][0], pf[i][1]);
            mma_f16(o[i][2 * w + 1], v1, pf[i][0], pf[i][1]);
          }
        }
      } else {
        uint32_t pf[kNT][2], rest[kNT][2];
#pragma unroll
        for (int i = 0; i < kNT; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t w = pack_bf16x2(s[i][2 * c], s[i][2 * c + 1]);
            rest[i][c] = transpose_8x8(pack_bf16x2(s[i][2 * c] - __uint_as_float(w << 16), s[i][2 * c + 1] - __uint_as_float(w & 0xFFFF0000u)));
            pf[i][c] = transpose_8x8(w);
          }
        uint32_t f_lo = 0, f_hi = 0;
        if constexpr (kFp8) {
          uint32_t f[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {  // code pattern = code * 2^-120; times 2^(126 + v - vr): the units of O, which carry 2^6
            const int key = 2 * tig + (y & 1) + 8 * (y >> 1);
            const uint32_t ve = __shfl_sync(0xFFFFFFFFu, e_now, 16 + key);
            const bool gone = key0 + key >= lim_max;
            f[y] = gone || (partly && ve == 255u) ? 0u
                   : ve == 255u ? 0x7FFFu
                                : static_cast<uint32_t>(max(0, static_cast<int>(ve) - static_cast<int>(vr) + 126 + 127)) << 7;
          }
          f_lo = f[0] | (f[1] << 16);
          f_hi = f[2] | (f[3] << 16);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t lo[2], hi[2];
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const int d = 2 * j + z;
            if constexpr (kFp8) {  // d = byte of the 16-byte piece; e4m3_pattern looks at bytes 1 and 3
              const int w = d >> 2, c = d & 3;
              const uint32_t pick = static_cast<uint32_t>(c << 4) | static_cast<uint32_t>((4 + c) << 12);
              lo[z] = mul_bf16x2(e4m3_pattern(__byte_perm(word_of(v[0], w), word_of(v[1], w), pick)), f_lo);
              hi[z] = mul_bf16x2(e4m3_pattern(__byte_perm(word_of(v[2], w), word_of(v[3], w), pick)), f_hi);
            } else {  // d = 8 * piece + dim in the piece
              const int x = d >> 3, w = (d & 7) >> 1;
              const uint32_t pick = (d & 1) ? 0x7632u : 0x5410u;
              lo[z] = __byte_perm(word_of(v[x], w), word_of(v[kVW + x], w), pick);
              hi[z] = __byte_perm(word_of(v[2 * kVW + x], w), word_of(v[3 * kVW + x], w), pick);
            }
          }
          const uint4 vf = make_uint4(lo[0], lo[1], hi[0], hi[1]);
#pragma unroll
          for (int i = 0; i < kNT; ++i) {
            mma_bf16(o[i][j], vf, pf[i][0], pf[i][1]);
            mma_bf16(o[i][j], vf, rest[i][0], rest[i][1]);
          }
        }
      }
      if (next < end_key) load_v(id, at);
    }

    // ---- the warps meet.  A lane holds, of rows 8 i + 2 tig + c, dims 8 gid + [0, 8) and 64 + 8 gid + [0, 8) (e4m3:
    //      16 gid + [0, 16)): dim d of its pieces is o[i][d / 2][2 (d % 2) + c]
    const float o_unit = kFp8 ? __uint_as_float(vr << 23) * (1.0f / 64.f) : 1.0f;  // no key at all: 0 * 0
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[i][c] += __shfl_xor_sync(0xFFFFFFFFu, l[i][c], x);
        const int r = 8 * i + 2 * tig + c;
        if (r < n_rows) {
#pragma unroll
          for (int d = 0; d < 16; d += 4)
            *reinterpret_cast<float4*>(&sm.o[warp][r][kFp8 ? 16 * gid + d : 64 * (d >> 3) + 8 * gid + (d & 7)]) =
                make_float4(o[i][d / 2][c] * o_unit, o[i][d / 2][2 + c] * o_unit, o[i][d / 2 + 1][c] * o_unit, o[i][d / 2 + 1][2 + c] * o_unit);
          if (gid == 0) {
            sm.m[warp][r] = m[i][c];
            sm.l[warp][r] = l[i][c];
          }
        }
      }
    __syncthreads();
    const bool whole = p.first && p.last;
    float* part = whole ? nullptr : part_slot(a, blockIdx.x, p.first);
    for (int x = threadIdx.x; x < n_rows * 16; x += kFewThreads) {  // 8 dims of a row per thread
      const int r = x >> 4, d0 = (x & 15) * 8;
      float top = kNoMax;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, sm.m[w][r]);
      float sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float f = ex2_approx(sm.m[w][r] - top);
        sum += sm.l[w][r] * f;
        const float4 v0 = *reinterpret_cast<const float4*>(&sm.o[w][r][d0]), v1 = *reinterpret_cast<const float4*>(&sm.o[w][r][d0 + 4]);
        acc[0] += v0.x * f; acc[1] += v0.y * f; acc[2] += v0.z * f; acc[3] += v0.w * f;
        acc[4] += v1.x * f; acc[5] += v1.y * f; acc[6] += v1.z * f; acc[7] += v1.w * f;
      }
      const int token = a.by_group(r0 + r), head = p.h * a.group + (r0 + r) - token * a.group;
      if (sm.poison) {  // rare: put back what was left out above, for the rows that see it
        const int end = min(key_limit(a, p.s, token), p.t1 << kFewKeyShift);
        for (int key = max(lim_min & ~15, p.t0 << kFewKeyShift); key < end; ++key)
          for (int d = 0; d < 8; ++d) {
            const float val = v_value<kFp8>(a, p.b, p.h, key, d0 + d);
            if (!isfinite(val)) acc[d] += val;
          }
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        uint4 w;
        w.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
        w.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
        w.z = pack_bf16x2(acc[4] * inv, acc[5] * inv);
        w.w = pack_bf16x2(acc[6] * inv, acc[7] * inv);
        *reinterpret_cast<uint4*>(a.o + (p.s.s0 + token) * a.o_stride_l + head * a.o_stride_h + d0) = w;
        if (a.lse && d0 == 0)
          a.lse[static_cast<long long>(head) * a.c.rows + p.s.s0 + token] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
      } else {
        *reinterpret_cast<float4*>(part + r * kCacheDim + d0) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        *reinterpret_cast<float4*>(part + r * kCacheDim + d0 + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
        if (d0 == 0) {
          part[kRows * kCacheDim + r] = top;
          part[kRows * kCacheDim + kRows + r] = sum;
        }
      }
    }
    if (threadIdx.x == 0 && p.first && !p.last)
      describe_join(a, sm.iter, sm.iter.item_base + a.set_up + item_tiles(a, p.s, p.it), n_rows, r0, p.s.s0, p.h);
    __syncthreads();  // everybody is done with this piece's shared memory
    if (threadIdx.x == 0) {
      sm.poison = 0;
      sm.more = sm.iter.next(a, sm.piece);
    }
  }
}

}  // namespace h3a
