// Attention of new rows over a paged K/V cache: what its kernels share (work distribution, partial results and the kernel
// that joins them).
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,  j < lengths[b], and with the causal mask j <= position of row i.
//
// Work.  An ITEM is a run of query rows of one sequence that share a K/V head (row r = token i * group + head in the
// group); it costs one unit per tile of keys plus one for its own set-up.  All items' units are laid end to end and cut
// into equal SHARES, one per CTA, whatever the lengths: a long sequence is spread over many SMs and many short ones share
// an SM.  An item that crosses a cut leaves fp32 partial results (O, running maximum, sum) in the workspace; a second small
// launch joins them in order of the keys, so results do not depend on timing.  A CTA has at most two such pieces (its
// first and its last), which bounds the workspace by the number of SMs, not by the batch.
#pragma once
#include "kv_cache.cuh"

namespace h3a {

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
  int key_shift;                     // log2 of the keys per tile
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
  return (key_limit(a, s, item_last_token(a, s, it)) + (1 << a.key_shift) - 1) >> a.key_shift;
}
// units of all the sequence's items of one K/V head
__device__ __forceinline__ long long head_units(const CacheAttnArgs& a, const AttnSeq& s) {
  if (!a.causal) return static_cast<long long>(s.n_items) * (1 + ((s.len + (1 << a.key_shift) - 1) >> a.key_shift));
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

}  // namespace h3a
