// Attention of new rows over a paged K/V cache: what its kernels share (work distribution, partial results and the kernel
// that joins them), and the kernel for few rows per K/V head.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,  j < lengths[b], and with the causal mask j <= position of row i.
//
// Work.  An ITEM is a run of query rows of one sequence that share a K/V head (row r = token i * group + head in the
// group); it costs one unit per 128-key tile plus one for its own set-up.  All items' units are laid end to end and cut
// into equal SHARES, one per CTA, whatever the lengths: a long sequence is spread over many SMs and many short ones share
// an SM.  An item that crosses a cut leaves fp32 partial results (O, running maximum, sum) in the workspace; a second small
// launch joins them in order of the keys, so results do not depend on timing.  A CTA has at most two such pieces (its
// first and its last), which bounds the workspace by the number of SMs, not by the batch.
#pragma once
#include "kv_cache.cuh"

namespace h3a {

constexpr int kKeyTile = 128;

struct CacheAttnArgs {
  CacheArgs c;                       // c.rows = query rows
  const uint8_t* q;                  // bf16 [rows, heads, 128]
  long long q_row_bytes, q_head_bytes;
  __nv_bfloat16* o;
  long long o_stride_l, o_stride_h;
  float* lse;                        // [heads, rows] or null
  int heads, group;                  // group = heads / kv_heads
  int causal;
  int item_rows;                     // rows per item (the kernel's tile)
  int item_tokens;                   // tokens per item, or 0: items are cut by rows, not by tokens
  float scale_log2;
  float* part;                       // [share][2][item_rows] x (128 + 2) fp32
  int* desc;                         // [share][4]: the item that a share begins and does not finish
  int min_share;                     // a share has at least this many units
  long long wait_ns;
};

struct AttnSeq {
  int s0, n, len, n_items;
};
__device__ __forceinline__ AttnSeq attn_seq(const CacheAttnArgs& a, int b) {
  const CacheSeq q = cache_seq(a.c, b);
  AttnSeq s;
  s.s0 = q.s0;
  s.n = q.n;
  s.len = q.len;
  s.n_items = a.item_tokens > 0 ? (q.n + a.item_tokens - 1) / a.item_tokens : (q.n * a.group + a.item_rows - 1) / a.item_rows;
  return s;
}
// keys that token i of the sequence sees
__device__ __forceinline__ int key_limit(const CacheAttnArgs& a, const AttnSeq& s, int i) {
  return a.causal ? max(0, min(s.len, s.len - s.n + i + 1)) : s.len;
}
__device__ __forceinline__ int item_last_token(const CacheAttnArgs& a, const AttnSeq& s, int it) {
  return min(s.n, a.item_tokens > 0 ? (it + 1) * a.item_tokens : ((it + 1) * a.item_rows + a.group - 1) / a.group) - 1;
}
__device__ __forceinline__ int item_tiles(const CacheAttnArgs& a, const AttnSeq& s, int it) {
  return (key_limit(a, s, item_last_token(a, s, it)) + kKeyTile - 1) / kKeyTile;
}
// units of all the sequence's items of one K/V head
__device__ __forceinline__ long long head_units(const CacheAttnArgs& a, const AttnSeq& s) {
  if (!a.causal) return static_cast<long long>(s.n_items) * (1 + (s.len + kKeyTile - 1) / kKeyTile);
  long long w = 0;
  for (int it = 0; it < s.n_items; ++it) w += 1 + item_tiles(a, s, it);
  return w;
}

struct ShareStart {     // in shared memory
  long long warp_sum[32];
  long long total;
  long long base;       // units before sequence `b`
  int b;
};

// A piece of an item: key tiles [t0, t1); `first` / `last`: it holds the item's first / last unit.
struct Piece {
  int b, h, it, t0, t1;
  bool first, last;
  AttnSeq s;
};

struct ShareIter {
  long long pos, end;     // units of this share still to do: [pos, end)
  long long item_base;    // first unit of the current item
  long long total;
  int n_shares;
  int b, h, it;
  AttnSeq s;

  __device__ __forceinline__ void skip_empty(const CacheAttnArgs& a) {
    while (s.n_items == 0 && b + 1 < a.c.n_seqs) s = attn_seq(a, ++b);
  }
  __device__ __forceinline__ bool next(const CacheAttnArgs& a, Piece& p) {
    if (pos >= end) return false;
    const int units = 1 + item_tiles(a, s, it);
    const int u0 = static_cast<int>(pos - item_base);
    const int u1 = static_cast<int>(min(static_cast<long long>(units), end - item_base));
    p.b = b;
    p.h = h;
    p.it = it;
    p.s = s;
    p.t0 = max(u0, 1) - 1;
    p.t1 = u1 - 1;
    p.first = u0 == 0;
    p.last = u1 == units;
    pos = item_base + u1;
    if (p.last) {
      item_base += units;
      if (++it == s.n_items) {
        it = 0;
        if (++h == a.c.kv_heads) {
          h = 0;
          if (b + 1 < a.c.n_seqs) {
            s = attn_seq(a, ++b);
            skip_empty(a);
          }
        }
      }
    }
    return true;
  }
};

__device__ __forceinline__ int n_shares_of(long long total, int grid, int min_share) {
  return static_cast<int>(max(1ll, min(static_cast<long long>(grid), total / min_share)));
}

// Executed by all threads of the block: finds where share `blockIdx.x` begins.  Every thread sums a run of sequences, the
// block scans the sums, and the thread whose run holds the share's first unit looks it up.
__device__ __forceinline__ ShareIter share_begin(const CacheAttnArgs& a, ShareStart* sh) {
  const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.c.n_seqs + nt - 1) / nt;
  const int b0 = min(a.c.n_seqs, tid * per), b1 = min(a.c.n_seqs, b0 + per);
  long long own = 0;
  for (int b = b0; b < b1; ++b) own += a.c.kv_heads * head_units(a, attn_seq(a, b));
  long long incl = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh->warp_sum[warp] = incl;
  if (tid == 0) sh->b = -1;
  __syncthreads();
  long long before = 0, total = 0;
  for (int w = 0; w < (nt >> 5); ++w) {
    const long long v = sh->warp_sum[w];
    before += w < warp ? v : 0;
    total += v;
  }
  before += incl - own;
  ShareIter s;
  s.total = total;
  s.n_shares = n_shares_of(total, gridDim.x, a.min_share);
  const int c = blockIdx.x;
  s.pos = c < s.n_shares ? total * c / s.n_shares : 0;
  s.end = c < s.n_shares ? total * (c + 1) / s.n_shares : 0;
  if (s.pos < s.end && before <= s.pos && s.pos < before + own) {
    long long base = before;
    for (int b = b0; b < b1; ++b) {
      const long long w = a.c.kv_heads * head_units(a, attn_seq(a, b));
      if (s.pos < base + w) {
        sh->b = b;
        sh->base = base;
        break;
      }
      base += w;
    }
  }
  __syncthreads();
  s.b = sh->b;
  s.h = s.it = 0;
  s.item_base = sh->base;
  if (s.b < 0) {  // an empty share
    s.end = s.pos;
    s.b = 0;
    return s;
  }
  s.s = attn_seq(a, s.b);
  const long long w = head_units(a, s.s);
  s.h = static_cast<int>((s.pos - s.item_base) / w);
  s.item_base += s.h * w;
  for (;;) {
    const int units = 1 + item_tiles(a, s.s, s.it);
    if (s.pos < s.item_base + units) break;
    s.item_base += units;
    ++s.it;
  }
  return s;
}

__device__ __forceinline__ float* part_slot(const CacheAttnArgs& a, int share, bool tail) {
  return a.part + (2ll * share + (tail ? 1 : 0)) * a.item_rows * (kCacheDim + 2);
}

// A page of the batch's table, brought into range (and reported) if it is not: what is read is then some other page's rows.
__device__ __forceinline__ int checked_page(const CacheAttnArgs& a, int b, int slot) {
  const int id = __ldg(a.c.pages + b * a.c.pages_stride + slot);
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.c.n_pages)) {
    report_cache(a.c, b);
    return 0;
  }
  return id;
}

constexpr float kNoMax = -3.0e38f;  // running maximum of a row that has seen no key: finite, so that differences stay numbers

// ---------------------------------------------------------------------------------------------------- joining
constexpr int kJoinRows = 4;  // a warp per row

// Block (share, y): rows [4 y, 4 y + 4) of the item that begins in the share and ends in a later one.
__global__ void __launch_bounds__(kJoinRows * 32) cache_attn_join_kernel(const CacheAttnArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the partial results are complete from here on
  if (a.c.status && *reinterpret_cast<volatile int*>(a.c.status) != 0) return;
  const int share = blockIdx.x;
  const int4 d = *reinterpret_cast<const int4*>(a.desc + 4 * share);  // sequence, head, item, last share
  if (d.x < 0) return;
  const AttnSeq s = attn_seq(a, d.x);
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.y * kJoinRows + (threadIdx.x >> 5);
  const int r0 = a.item_tokens > 0 ? d.z * a.item_tokens * a.group : d.z * a.item_rows;
  const int n_rows = min(s.n * a.group - r0, a.item_tokens > 0 ? a.item_tokens * a.group : a.item_rows);
  if (r >= n_rows) return;
  // parts of the row: the tail slot of this share, then the head slots of the next ones
  const int n_parts = d.w - share + 1;
  auto slot = [&](int i) { return part_slot(a, share + i, i == 0); };
  auto stat = [&](int i, int which) { return slot(i)[a.item_rows * kCacheDim + which * a.item_rows + r]; };
  float m = kNoMax;
  for (int i = lane; i < n_parts; i += 32) m = fmaxf(m, stat(i, 0));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int i = 0; i < n_parts; ++i) {
    const float w = ex2_approx(stat(i, 0) - m);
    const float4 v = *reinterpret_cast<const float4*>(slot(i) + r * kCacheDim + 4 * lane);
    l += stat(i, 1) * w;
    acc.x += v.x * w;
    acc.y += v.y * w;
    acc.z += v.z * w;
    acc.w += v.w * w;
  }
  const int row = r0 + r, token = s.s0 + row / a.group, head = d.y * a.group + row % a.group;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint2 w;
  w.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  w.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(a.o + token * a.o_stride_l + head * a.o_stride_h + 4 * lane) = w;
  if (a.lse && lane == 0)
    a.lse[static_cast<long long>(head) * a.c.rows + token] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// ---------------------------------------------------------------------------------------------------- few rows
// Up to 16 rows per item.  HBM-bound: the cache is read once, 2 x 256 B (2 x 129 B) per key and head, for 4 x 16 x 128
// multiply-adds.  So no shared memory and no tensor-memory round trip: a warp takes 16 keys of every tile, loads them
// straight into the register fragments of the warp-level MMA (m16n8k16, bf16) and keeps the next tile's loads in flight
// while it works.  The MMA leaves the order of the contraction free: for Q K^T a lane's four 16-byte pieces of a K row
// are the dims it contributes to the k-steps (Q is permuted alike, once); for P V it loads 16-byte pieces of the four
// keys its fragment needs, paired by byte permutes, and the output columns come out permuted, 16 (32) consecutive dims
// per lane.  Eight warps with their own running maximum and sum meet in shared memory once per piece.
constexpr int kFewRows = 16;
constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewSmemBytes = kFewWarps * kFewRows * (kCacheDim + 4) * 4 + kFewWarps * kFewRows * 2 * 4 + 8 * 32 * 16;

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3,
                                         const uint32_t b0, const uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 keys of one head as loaded: K rows 8 u + lane / 4 (u = 0, 1), V rows 2 (lane % 4) + {0, 1, 8, 9}
template <bool kFp8>
struct KeyBlock {
  uint4 k[kFp8 ? 4 : 8];  // [u][piece]
  uint4 v[kFp8 ? 4 : 8];  // [key][piece]
  uint32_t e;             // lanes 0-15: exponent byte of K row `lane`; lanes 16-31: of V row `lane - 16`
};

__device__ __forceinline__ bool non_finite2(uint32_t w) {
  return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}
__device__ __forceinline__ uint32_t finite_or_zero2(uint32_t w) {
  if ((w & 0x7F80u) == 0x7F80u) w &= 0xFFFF0000u;
  if ((w & 0x7F800000u) == 0x7F800000u) w &= 0x0000FFFFu;
  return w;
}
// value of dim `d` of a V row, whatever the cache holds it in
template <bool kFp8>
__device__ __forceinline__ float v_value(const CacheAttnArgs& a, int b, int h, int key, int d) {
  const int slot = key / a.c.page_size, at = key - slot * a.c.page_size;
  const long long id = checked_page(a, b, slot);
  const uint8_t* row = a.c.pool[1] + id * a.c.page_bytes[1] + at * a.c.token_bytes[1] + h * a.c.head_bytes[1];
  if constexpr (kFp8) {
    const uint32_t e = a.c.exps[1][id * a.c.exp_page[1] + at * a.c.exp_token[1] + h * a.c.exp_head[1]];
    const uint32_t w = mul_bf16x2(mul_bf16x2(e4m3_pattern(static_cast<uint32_t>(row[d]) << 8), e4m3_factor(e)), e4m3_factor2(e));
    return __uint_as_float(w << 16);
  } else {
    return __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[d]) << 16);
  }
}

template <bool kFp8>
__global__ void __launch_bounds__(kFewThreads, 1) cache_attn_few_kernel(const CacheAttnArgs a) {
  extern __shared__ float few_smem[];
  __shared__ ShareStart start;
  __shared__ int poison_s[2];  // per piece, in turn: some V value that only part of the item's rows see is not finite
  if (a.c.status && *reinterpret_cast<volatile int*>(a.c.status) != 0) return;
  constexpr int kORow = kCacheDim + 4;  // padded row of O in shared memory
  float* o_s = few_smem;                                        // [warp][16][kORow]
  float* m_s = few_smem + kFewWarps * kFewRows * kORow;         // [warp][16]
  float* l_s = m_s + kFewWarps * kFewRows;                      // [warp][16]
  uint4* q_s = reinterpret_cast<uint4*>(l_s + kFewWarps * kFewRows);  // [k-step][lane]: Q fragments (registers are for K and V)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;

  ShareIter iter = share_begin(a, &start);
  if (threadIdx.x == 0) {
    poison_s[0] = 0;
    a.desc[4 * blockIdx.x] = -1;
  }
  __syncthreads();
  Piece p;
  for (int turn = 0; iter.next(a, p); turn ^= 1) {
    int& poison = poison_s[turn];
    if (threadIdx.x == 0) poison_s[turn ^ 1] = 0;  // last read in the previous piece, next written in the next one
    const int r0 = p.it * kFewRows;
    const int n_rows = min(kFewRows, p.s.n * a.group - r0);
    // ---- Q fragments: rows gid and gid + 8, dims in the order of the K loads below; warp x loads piece x of all rows
    int lim[2];
    {
      uint4 w[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int r = gid + 8 * y;
        const bool have = r < n_rows;
        const int token = have ? (r0 + r) / a.group : 0;
        const int head = p.h * a.group + (r0 + r) - token * a.group;
        lim[y] = have ? key_limit(a, p.s, token) : 0;
        // bf16: piece x = dims 32 x + 8 tig + [0, 8); e4m3: pieces 2 c, 2 c + 1 = dims 64 c + 16 tig + [0, 16)
        const int dim = kFp8 ? 64 * (warp >> 1) + 16 * tig + 8 * (warp & 1) : 32 * warp + 8 * tig;
        w[y] = make_uint4(0, 0, 0, 0);
        if (warp < 4 && have) w[y] = __ldg(reinterpret_cast<const uint4*>(a.q + (p.s.s0 + token) * a.q_row_bytes + head * a.q_head_bytes + 2 * dim));
      }
      if (warp < 4) {
        q_s[2 * warp * 32 + lane] = make_uint4(w[0].x, w[1].x, w[0].y, w[1].y);
        q_s[(2 * warp + 1) * 32 + lane] = make_uint4(w[0].z, w[1].z, w[0].w, w[1].w);
      }
    }
    __syncthreads();
    const int lim_min = key_limit(a, p.s, r0 / a.group);
    const int lim_max = key_limit(a, p.s, item_last_token(a, p.s, p.it));

    float o[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m[2] = {kNoMax, kNoMax}, l[2] = {0.f, 0.f};

    // the warp's 16 keys of tile t: none, if they lie behind the last key any row sees
    auto has = [&](int t) { return t < p.t1 && t * kKeyTile + warp * 16 < lim_max; };
    auto page_of = [&](int t) { return checked_page(a, p.b, (t * kKeyTile + warp * 16) / a.c.page_size); };
    auto load = [&](KeyBlock<kFp8>& blk, int t, long long id) {
      const int key0 = t * kKeyTile + warp * 16;
      const int at = key0 % a.c.page_size;
      const uint8_t* kb = a.c.pool[0] + id * a.c.page_bytes[0] + at * a.c.token_bytes[0] + p.h * a.c.head_bytes[0];
      const uint8_t* vb = a.c.pool[1] + id * a.c.page_bytes[1] + at * a.c.token_bytes[1] + p.h * a.c.head_bytes[1];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int x = 0; x < (kFp8 ? 2 : 4); ++x)
          blk.k[u * (kFp8 ? 2 : 4) + x] = ldg_stream(kb + (8 * u + gid) * a.c.token_bytes[0] + 64 * x + 16 * tig);
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int x = 0; x < (kFp8 ? 1 : 2); ++x)
          blk.v[y * (kFp8 ? 1 : 2) + x] = ldg_stream(vb + (2 * tig + (y & 1) + 8 * (y >> 1)) * a.c.token_bytes[1] + 128 * x + 16 * gid);
      if constexpr (kFp8) {
        const int x = lane >> 4;
        blk.e = __ldg(a.c.exps[x] + id * a.c.exp_page[x] + (at + (lane & 15)) * a.c.exp_token[x] + p.h * a.c.exp_head[x]);
      }
    };
    auto compute = [&](KeyBlock<kFp8>& blk, int t) {
      const int key0 = t * kKeyTile + warp * 16;
      // ---- S = Q K^T
      float s[2][4];
      uint32_t f[2], f2[2];
      bool two_k = false;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
        if constexpr (kFp8) {
          const uint32_t e = __shfl_sync(0xFFFFFFFFu, blk.e, 8 * u + gid);
          f[u] = e4m3_factor(e) * 0x10001u;
          f2[u] = e4m3_factor2(e) * 0x10001u;
          two_k |= e > kOneStepExp;
        }
      }
      two_k = kFp8 && __any_sync(0xFFFFFFFFu, two_k);
#pragma unroll
      for (int x = 0; x < 8; ++x) {  // k-step
        const uint4 qf = q_s[x * 32 + lane];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t b0, b1;
          if constexpr (kFp8) {
            const uint4& piece = blk.k[2 * u + (x >> 2)];
            const uint32_t w = (x & 3) == 0 ? piece.x : (x & 3) == 1 ? piece.y : (x & 3) == 2 ? piece.z : piece.w;
            b0 = mul_bf16x2(e4m3_pattern(__byte_perm(w, 0, 0x1404)), f[u]);
            b1 = mul_bf16x2(e4m3_pattern(__byte_perm(w, 0, 0x3424)), f[u]);
            if (two_k) {
              b0 = mul_bf16x2(b0, f2[u]);
              b1 = mul_bf16x2(b1, f2[u]);
            }
          } else {
            const uint4& piece = blk.k[4 * u + (x >> 1)];
            b0 = (x & 1) ? piece.z : piece.x;
            b1 = (x & 1) ? piece.w : piece.y;
          }
          mma_bf16(s[u], qf.x, qf.y, qf.z, qf.w, b0, b1);
        }
      }
      // ---- softmax: s[u][0, 1] are row gid, s[u][2, 3] row gid + 8; keys 8 u + 2 tig + {0, 1}
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int y = 0; y < 4; ++y) s[u][y] *= a.scale_log2;
      const bool partly = key0 + 16 > lim_min;  // some row does not see some key (or a row is not there at all)
      if (partly) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if (key0 + 8 * u + 2 * tig + (y & 1) >= lim[y >> 1]) s[u][y] = -INFINITY;
      }
      float top[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        top[y] = fmaxf(fmaxf(s[0][2 * y], s[0][2 * y + 1]), fmaxf(s[1][2 * y], s[1][2 * y + 1]));
        top[y] = fmaxf(top[y], __shfl_xor_sync(0xFFFFFFFFu, top[y], 1));
        top[y] = fmaxf(top[y], __shfl_xor_sync(0xFFFFFFFFu, top[y], 2));
      }
      // O is rescaled only when a row's maximum grows by more than 2^8: terms stay far inside fp32 until then
      if (__any_sync(0xFFFFFFFFu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f)) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float m_new = fmaxf(m[y], top[y]);
          const float f = ex2_approx(m[y] - m_new);
          m[y] = m_new;
          l[y] *= f;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            o[j][2 * y] *= f;
            o[j][2 * y + 1] *= f;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          s[u][y] = ex2_approx(s[u][y] - m[y >> 1]);
          l[y >> 1] += s[u][y];
        }
      // P in bf16: one rounding per term, of at most 2^-9 of it; the row sum keeps the unrounded terms
      const uint32_t p0 = pack_bf16x2(s[0][0], s[0][1]), p1 = pack_bf16x2(s[0][2], s[0][3]);
      const uint32_t p2 = pack_bf16x2(s[1][0], s[1][1]), p3 = pack_bf16x2(s[1][2], s[1][3]);
      // ---- O += P V.  P is 0 where a key is masked, so V must be finite there: rows behind the sequence's last key may
      //      hold anything and count as zeros; a value that some of the item's rows see and others do not counts as zero
      //      if it is not finite, and is put back at the end for the rows that see it.
      uint32_t f_lo = 0, f_hi = 0, g_lo = 0, g_hi = 0;
      bool two = false;
      if constexpr (kFp8) {
        uint32_t f[4], g[4];
        bool bad = false;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int key = 2 * tig + (y & 1) + 8 * (y >> 1);
          const uint32_t e = __shfl_sync(0xFFFFFFFFu, blk.e, 16 + key);
          const bool gone = key0 + key >= lim_max;
          const bool poisoned = partly && e == 255u;
          bad |= poisoned && !gone;
          f[y] = gone || poisoned ? 0u : e4m3_factor(e);
          g[y] = e4m3_factor2(e);
          two |= e > kOneStepExp;
        }
        if (bad) poison = 1;
        two = __any_sync(0xFFFFFFFFu, two);
        f_lo = f[0] | (f[1] << 16);
        f_hi = f[2] | (f[3] << 16);
        g_lo = g[0] | (g[1] << 16);
        g_hi = g[2] | (g[3] << 16);
      } else if (partly) {
        bool bad = false;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const bool gone = key0 + 2 * tig + (y & 1) + 8 * (y >> 1) >= lim_max;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint4& w = blk.v[2 * y + x];
            if (gone) w = make_uint4(0, 0, 0, 0);
            bad |= non_finite2(w.x) || non_finite2(w.y) || non_finite2(w.z) || non_finite2(w.w);
            w = make_uint4(finite_or_zero2(w.x), finite_or_zero2(w.y), finite_or_zero2(w.z), finite_or_zero2(w.w));
          }
        }
        if (bad) poison = 1;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        uint32_t b0, b1;
        if constexpr (kFp8) {  // j = byte of the 16-byte piece
          const int w = j >> 2, c = j & 3;
          const uint32_t x0 = w == 0 ? blk.v[0].x : w == 1 ? blk.v[0].y : w == 2 ? blk.v[0].z : blk.v[0].w;
          const uint32_t x1 = w == 0 ? blk.v[1].x : w == 1 ? blk.v[1].y : w == 2 ? blk.v[1].z : blk.v[1].w;
          const uint32_t x2 = w == 0 ? blk.v[2].x : w == 1 ? blk.v[2].y : w == 2 ? blk.v[2].z : blk.v[2].w;
          const uint32_t x3 = w == 0 ? blk.v[3].x : w == 1 ? blk.v[3].y : w == 2 ? blk.v[3].z : blk.v[3].w;
          // bytes 1 and 3 of the result are what e4m3_pattern looks at: byte c of each key's word
          const uint32_t pick = static_cast<uint32_t>(c << 4) | static_cast<uint32_t>((4 + c) << 12);
          b0 = mul_bf16x2(e4m3_pattern(__byte_perm(x0, x1, pick)), f_lo);
          b1 = mul_bf16x2(e4m3_pattern(__byte_perm(x2, x3, pick)), f_hi);
          if (two) {
            b0 = mul_bf16x2(b0, g_lo);
            b1 = mul_bf16x2(b1, g_hi);
          }
        } else {  // j = 8 * piece + dim in the piece
          const int x = j >> 3, w = (j & 7) >> 1;
          const uint32_t x0 = w == 0 ? blk.v[x].x : w == 1 ? blk.v[x].y : w == 2 ? blk.v[x].z : blk.v[x].w;
          const uint32_t x1 = w == 0 ? blk.v[2 + x].x : w == 1 ? blk.v[2 + x].y : w == 2 ? blk.v[2 + x].z : blk.v[2 + x].w;
          const uint32_t x2 = w == 0 ? blk.v[4 + x].x : w == 1 ? blk.v[4 + x].y : w == 2 ? blk.v[4 + x].z : blk.v[4 + x].w;
          const uint32_t x3 = w == 0 ? blk.v[6 + x].x : w == 1 ? blk.v[6 + x].y : w == 2 ? blk.v[6 + x].z : blk.v[6 + x].w;
          const uint32_t pick = (j & 1) ? 0x7632u : 0x5410u;
          b0 = __byte_perm(x0, x1, pick);
          b1 = __byte_perm(x2, x3, pick);
        }
        mma_bf16(o[j], p0, p1, p2, p3, b0, b1);
      }
    };

    {
      KeyBlock<kFp8> ba, bb;
      int t = p.t0;
      long long id = has(t) ? page_of(t) : 0;
      if (has(t)) load(ba, t, id);
      id = has(t + 1) ? page_of(t + 1) : 0;
      while (has(t)) {
        if (has(t + 1)) load(bb, t + 1, id);
        id = has(t + 2) ? page_of(t + 2) : 0;
        compute(ba, t);
        ++t;
        if (!has(t)) break;
        if (has(t + 1)) load(ba, t + 1, id);
        id = has(t + 2) ? page_of(t + 2) : 0;
        compute(bb, t);
        ++t;
      }
    }

    // ---- the warps meet.  A lane holds, of row gid (+ 8), 16 dims from 16 tig and from 64 + 16 tig (e4m3: 32 from 32 tig):
    //      column 2 tig + (y & 1) of n-tile j is that row's dim j of the piece of lane group 2 tig + (y & 1)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      l[y] += __shfl_xor_sync(0xFFFFFFFFu, l[y], 1);
      l[y] += __shfl_xor_sync(0xFFFFFFFFu, l[y], 2);
      const int r = gid + 8 * y;
      float* row = o_s + (warp * kFewRows + r) * kORow;
      if (r < n_rows) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if constexpr (kFp8) {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(row + (2 * tig + c) * 16 + j) =
                  make_float4(o[j][2 * y + c], o[j + 1][2 * y + c], o[j + 2][2 * y + c], o[j + 3][2 * y + c]);
          } else {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(row + 64 * (j >> 3) + (2 * tig + c) * 8 + (j & 7)) =
                  make_float4(o[j][2 * y + c], o[j + 1][2 * y + c], o[j + 2][2 * y + c], o[j + 3][2 * y + c]);
          }
        }
        if (tig == 0) {
          m_s[warp * kFewRows + r] = m[y];
          l_s[warp * kFewRows + r] = l[y];
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
      for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, m_s[w * kFewRows + r]);
      float sum = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float f = ex2_approx(m_s[w * kFewRows + r] - top);
        sum += l_s[w * kFewRows + r] * f;
        const float* src = o_s + (w * kFewRows + r) * kORow + d0;
        const float4 v0 = *reinterpret_cast<const float4*>(src), v1 = *reinterpret_cast<const float4*>(src + 4);
        acc[0] += v0.x * f; acc[1] += v0.y * f; acc[2] += v0.z * f; acc[3] += v0.w * f;
        acc[4] += v1.x * f; acc[5] += v1.y * f; acc[6] += v1.z * f; acc[7] += v1.w * f;
      }
      const int token = (r0 + r) / a.group, head = p.h * a.group + (r0 + r) - token * a.group;
      if (poison) {  // rare: put back what was left out above, for the rows that see it
        const int end = min(key_limit(a, p.s, token), p.t1 * kKeyTile);
        for (int key = max(lim_min & ~15, p.t0 * kKeyTile); key < end; ++key)
          for (int d = 0; d < 8; ++d) {
            const float v = v_value<kFp8>(a, p.b, p.h, key, d0 + d);
            if (!isfinite(v)) acc[d] += v;
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
          part[kFewRows * kCacheDim + r] = top;
          part[kFewRows * kCacheDim + kFewRows + r] = sum;
        }
      }
    }
    if (threadIdx.x == 0 && p.first && !p.last) {  // the item goes on in later shares: say where it ends
      const long long item_end = iter.item_base + 1 + item_tiles(a, p.s, p.it);
      const int last = static_cast<int>((item_end * iter.n_shares + iter.total - 1) / iter.total) - 1;
      *reinterpret_cast<int4*>(a.desc + 4 * blockIdx.x) = make_int4(p.b, p.h, p.it, last);
    }
    __syncthreads();
  }
}

}  // namespace h3a
