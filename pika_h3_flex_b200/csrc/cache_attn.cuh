// Attention of new rows over a paged K/V cache: what its kernels share (work distribution, partial results and the kernel
// that joins them).
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,  j < lengths[b], and with the causal mask j <= position of row i.
//
// Work.  An ITEM is a run of query rows of one sequence that share a K/V head (row r = token i * group + head in the
// group); it costs one unit per tile of keys plus `set_up`.  All items' units are laid end to end and cut
// into equal SHARES, one per CTA, whatever the lengths: a long sequence is spread over many SMs and many short ones share
// an SM.  An item that crosses a cut leaves fp32 partial results (O, running maximum, sum) in the workspace; a second small
// launch joins them in order of the keys, so results do not depend on timing.  A CTA has at most two such pieces (its
// first and its last), which bounds the workspace by the number of SMs, not by the batch.
//
// Laid end to end, neighbouring CTAs are at different keys of different heads at any moment, and where K and V do not fit
// L2 every CTA fetches them from HBM for itself (40 heads of 49,384 keys: 18 of the 19 GB that the items read).  So where
// all items cost the same and there are more of them than CTAs (one sequence without a causal mask), whole items are dealt
// out in rounds, the CTAs of a round walking the same few heads' keys in step, and only the last, partial round is cut.
#pragma once
#include "kv_cache.cuh"

namespace h3a {

struct CacheAttnArgs {
  CacheArgs c;                       // c.rows = query rows
  const uint8_t* q;                  // bf16 [rows, heads, 128]
  long long q_row_bytes, q_head_bytes;
  __nv_bfloat16* o;
  long long o_stride_l, o_stride_h;
  int o_sectors;                     // rows of o begin at multiples of 32 bytes
  float* lse;                        // [heads, rows] or null
  int heads, group;                  // group = heads / kv_heads
  FastDiv by_group, by_item_tokens, by_item_rows;
  int causal;
  int item_rows;                     // rows per item (the kernel's tile)
  int item_tokens;                   // tokens per item, or 0: items are cut by rows, not by tokens
  int key_shift;                     // log2 of the keys per tile
  float scale_log2;
  float* part;                       // [share][2][item_rows] x (128 + 2) fp32
  int* desc;                         // [share][kDescInts]: the item that a share begins and does not finish
  int shares;                        // CTAs of the kernel
  int set_up;                        // units that an item costs beside one per tile
  int share_shift;                   // a share has at least 2^this units
  uint32_t wait_units;               // longest wait, in 1,024 ns
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
  s.n_items = a.item_tokens > 0 ? a.by_item_tokens(q.n + a.item_tokens - 1) : a.by_item_rows(q.n * a.group + a.item_rows - 1);
  return s;
}
// keys that token i of the sequence sees
__device__ __forceinline__ int key_limit(const CacheAttnArgs& a, const AttnSeq& s, int i) {
  return a.causal ? max(0, min(s.len, s.len - s.n + i + 1)) : s.len;
}
__device__ __forceinline__ int item_last_token(const CacheAttnArgs& a, const AttnSeq& s, int it) {
  return min(s.n, a.item_tokens > 0 ? (it + 1) * a.item_tokens : a.by_group((it + 1) * a.item_rows + a.group - 1)) - 1;
}
__device__ __forceinline__ int item_tiles(const CacheAttnArgs& a, const AttnSeq& s, int it) {
  return (key_limit(a, s, item_last_token(a, s, it)) + (1 << a.key_shift) - 1) >> a.key_shift;
}
// units of all the sequence's items of one K/V head
__device__ __forceinline__ long long head_units(const CacheAttnArgs& a, const AttnSeq& s) {
  if (!a.causal) return static_cast<long long>(s.n_items) * (a.set_up + ((s.len + (1 << a.key_shift) - 1) >> a.key_shift));
  long long w = 0;
  for (int it = 0; it < s.n_items; ++it) w += a.set_up + item_tiles(a, s, it);
  return w;
}

struct ShareStart {     // in shared memory
  long long warp_sum[32];
  long long total;
  long long base;       // units before sequence `b`
  int b;
};

// A piece of an item: key tiles [t0, t1); `first` / `last`: it holds the item's first / last tile.
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
  int whole, whole_item;  // whole items dealt to this CTA and not yet begun; number of the next one

  __device__ __forceinline__ void skip_empty(const CacheAttnArgs& a) {
    while (s.n_items == 0 && b + 1 < a.c.n_seqs) s = attn_seq(a, ++b);
  }
  __device__ __forceinline__ bool next(const CacheAttnArgs& a, Piece& p) {
    if (whole > 0) {
      p.b = b;
      p.h = whole_item / s.n_items;
      p.it = whole_item - p.h * s.n_items;
      p.s = s;
      p.t0 = 0;
      p.t1 = item_tiles(a, s, p.it);
      p.first = p.last = true;
      whole_item += gridDim.x;
      --whole;
      return true;
    }
    if (pos >= end) return false;
    const int units = a.set_up + item_tiles(a, s, it);
    const int u0 = static_cast<int>(pos - item_base);
    const int u1 = static_cast<int>(min(static_cast<long long>(units), end - item_base));
    p.b = b;
    p.h = h;
    p.it = it;
    p.s = s;
    pos = item_base + u1;
    p.t0 = max(u0 - a.set_up, 0);
    p.t1 = u1 - a.set_up;
    p.first = p.t0 == 0;
    p.last = u1 == units;
    if (p.t1 <= 0 && !p.last) return false;  // the share ends before the item's first tile: the next one begins it
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

// a / b, in 32 bits where they fit: the 64-bit division is a loop of some 70 instructions
__device__ __forceinline__ long long div_units(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}
// which units share c has: [total c / n, total (c + 1) / n)
__device__ __forceinline__ void share_range(const CacheAttnArgs& a, ShareIter& s) {
  s.n_shares = static_cast<int>(max(1ll, min(static_cast<long long>(gridDim.x), s.total >> a.share_shift)));
  const int c = blockIdx.x;
  const long long q = div_units(s.total, s.n_shares);
  const uint32_t r = static_cast<uint32_t>(s.total - q * s.n_shares), n = s.n_shares;
  s.pos = c < s.n_shares ? q * c + r * c / n : 0;
  s.end = c < s.n_shares ? q * (c + 1) + r * (c + 1) / n : 0;
}
// the share's first item, given its first sequence and the units before that
__device__ __forceinline__ void share_item(const CacheAttnArgs& a, ShareIter& s, long long head_total) {
  s.h = static_cast<int>(div_units(s.pos - s.item_base, head_total));
  s.item_base += s.h * head_total;
  s.it = 0;
  if (!a.causal) {  // items of equal length
    const int units = a.set_up + item_tiles(a, s.s, 0);
    s.it = static_cast<int>(div_units(s.pos - s.item_base, units));
    s.item_base += static_cast<long long>(s.it) * units;
    return;
  }
  for (;;) {
    const int units = a.set_up + item_tiles(a, s.s, s.it);
    if (s.pos < s.item_base + units) break;
    s.item_base += units;
    ++s.it;
  }
}

// Executed by all threads of the block: finds where share `blockIdx.x` begins, the same in every thread.  Up to 32
// sequences every warp does it by itself, one sequence per lane, without a barrier: a single token's call is over in a few
// microseconds.  More sequences: every thread sums a run of them, the block scans the sums, and the thread whose run holds
// the share's first unit looks it up.
__device__ __forceinline__ ShareIter share_begin(const CacheAttnArgs& a, ShareStart* sh) {
  const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  ShareIter s;
  s.whole = s.whole_item = 0;
  if (a.c.n_seqs == 1 && !a.causal && a.item_tokens > 0) {
    s.b = 0;
    s.s = attn_seq(a, 0);
    const int n_items = s.s.n_items * a.c.kv_heads, units = a.set_up + item_tiles(a, s.s, 0);
    s.whole = n_items / gridDim.x;
    s.whole_item = blockIdx.x;
    const int dealt = s.whole * gridDim.x;
    s.total = static_cast<long long>(n_items - dealt) * units;
    share_range(a, s);
    const int ahead = static_cast<int>(div_units(s.pos, units));  // items of the last round before this share's first
    s.item_base = static_cast<long long>(ahead) * units;
    s.h = s.s.n_items > 0 ? (dealt + ahead) / s.s.n_items : 0;
    s.it = dealt + ahead - s.h * s.s.n_items;
    return s;
  }
  if (a.c.n_seqs <= 32) {
    AttnSeq q{0, 0, 0, 0};
    long long head_total = 0;
    if (lane < a.c.n_seqs) {
      q = attn_seq(a, lane);
      head_total = head_units(a, q);
    }
    const long long own = a.c.kv_heads * head_total;
    long long incl = own;
    for (int o = 1; o < a.c.n_seqs; o <<= 1) {
      const long long v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += v;
    }
    s.total = __shfl_sync(0xFFFFFFFFu, incl, a.c.n_seqs - 1);
    share_range(a, s);
    const uint32_t here = __ballot_sync(0xFFFFFFFFu, s.pos < s.end && incl - own <= s.pos && s.pos < incl);
    const int b = max(0, __ffs(here) - 1);
    s.b = b;
    s.h = s.it = 0;
    s.s.s0 = __shfl_sync(0xFFFFFFFFu, q.s0, b);
    s.s.n = __shfl_sync(0xFFFFFFFFu, q.n, b);
    s.s.len = __shfl_sync(0xFFFFFFFFu, q.len, b);
    s.s.n_items = __shfl_sync(0xFFFFFFFFu, q.n_items, b);
    s.item_base = __shfl_sync(0xFFFFFFFFu, incl - own, b);
    head_total = __shfl_sync(0xFFFFFFFFu, head_total, b);
    if (here == 0) s.end = s.pos;  // an empty share
    else share_item(a, s, head_total);
    return s;
  }
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
  s.total = total;
  share_range(a, s);
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
  share_item(a, s, head_units(a, s.s));
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

// the e4m3 codes in bytes 0 and 1 of w as fp16
__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_high_to_f16x2(uint32_t w) {  // bytes 2 and 3
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// 2^e, within the range of normal numbers
__device__ __forceinline__ float pow2_float(int e) { return __uint_as_float(static_cast<uint32_t>(max(-126, min(e, 127)) + 127) << 23); }

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
  const int slot = a.c.by_page(key), at = key - slot * a.c.page_size;
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

// Least factor from S to logits.  A row of zeros in Q against rows of zeros in K has one that underflows, and a masked logit
// times 0 is no longer -inf but NaN; with this one such a row's own logits, at most 2^21 times it, are still 0.
constexpr float kLeastUnit = 1.17549435e-38f;  // 2^-126

// lets the launch of the kernel that follows (the join) begin; it waits for this one's results itself
__device__ __forceinline__ void allow_next_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---------------------------------------------------------------------------------------------------- joining
constexpr int kJoinRows = 4;  // a warp per row
constexpr int kDescInts = 8;  // parts (0: no such item), rows, first row (token * group + head in the group), sequence's first packed row, K/V head
// The item that begins in this share goes on in later ones, up to the one that holds unit item_end - 1.
__device__ __forceinline__ void describe_join(const CacheAttnArgs& a, const ShareIter& s, long long item_end, int n_rows, int r0, int s0, int h) {
  const int last = static_cast<int>(div_units(item_end * s.n_shares + s.total - 1, s.total)) - 1;
  int* d = a.desc + kDescInts * blockIdx.x;
  *reinterpret_cast<int4*>(d) = make_int4(last - static_cast<int>(blockIdx.x) + 1, n_rows, r0, s0);
  d[4] = h;
}

// A warp's share of a row's parts, first_part, first_part + stride, ... kJoinParts at a time, whose loads wait for nothing
// but the item's description: with the parts one after the other a row of 37 took 29 us.
struct JoinRow {
  float m, l;
  float4 acc;  // dims 4 lane + [0, 4)
};
template <int kJoinParts>
__device__ __forceinline__ JoinRow join_parts(const CacheAttnArgs& a, int share, int r, int n_parts, int first_part, int stride) {
  const int lane = threadIdx.x & 31;
  // parts of the row: the tail slot of its first share, then the head slots of the next ones
  const long long slot = 2ll * a.item_rows * (kCacheDim + 2);
  const float* first = part_slot(a, share, true);
  const float* next = part_slot(a, share, false);  // + i slots for part i > 0
  JoinRow row{kNoMax, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int i0 = first_part; i0 < n_parts; i0 += stride) {
    const int n = min(kJoinParts, n_parts - i0);
    float4 v[kJoinParts];
#pragma unroll
    for (int i = 0; i < kJoinParts; ++i)
      if (i < n) v[i] = *reinterpret_cast<const float4*>((i0 + i == 0 ? first : next + (i0 + i) * slot) + r * kCacheDim + 4 * lane);
    float mi = kNoMax, li = 0.f;
    if (lane < n) {
      const float* st = (i0 + lane == 0 ? first : next + (i0 + lane) * slot) + a.item_rows * kCacheDim + r;
      mi = st[0];
      li = st[a.item_rows];
    }
    float top = mi;
#pragma unroll
    for (int o = kJoinParts / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    top = __shfl_sync(0xFFFFFFFFu, top, 0);
    const float m_new = fmaxf(row.m, top), f = ex2_approx(row.m - m_new), wi = ex2_approx(mi - m_new);
    row.m = m_new;
    row.l *= f;
    row.acc = make_float4(row.acc.x * f, row.acc.y * f, row.acc.z * f, row.acc.w * f);
#pragma unroll
    for (int i = 0; i < kJoinParts; ++i)
      if (i < n) {
        const float w = __shfl_sync(0xFFFFFFFFu, wi, i);
        row.l += w * __shfl_sync(0xFFFFFFFFu, li, i);
        row.acc.x += v[i].x * w;
        row.acc.y += v[i].y * w;
        row.acc.z += v[i].z * w;
        row.acc.w += v[i].w * w;
      }
  }
  return row;
}
// row `row` (token * group + head in the group) of the sequence whose first packed row is s0
__device__ __forceinline__ void store_joined(const CacheAttnArgs& a, const JoinRow& x, int row, int s0, int kv_head) {
  const int lane = threadIdx.x & 31;
  const int i = a.by_group(row), token = s0 + i, head = kv_head * a.group + row - i * a.group;
  const float inv = x.l == 0.f ? 0.f : 1.0f / x.l;
  uint2 w;
  w.x = pack_bf16x2(x.acc.x * inv, x.acc.y * inv);
  w.y = pack_bf16x2(x.acc.z * inv, x.acc.w * inv);
  *reinterpret_cast<uint2*>(a.o + token * a.o_stride_l + head * a.o_stride_h + 4 * lane) = w;
  if (a.lse && lane == 0)
    a.lse[static_cast<long long>(head) * a.c.rows + token] = x.l == 0.f ? -INFINITY : (x.m + log2f(x.l)) * 0.6931471805599453f;
}

// Block (share, y): rows 4 y + [0, 4), and so on, of the item that begins in the share and ends in a later one, a warp per
// row.  The kernel is a few dependent loads long, so its launch overlaps the kernel before it, and everything it has to know
// about the item is in the description.  16 parts at a time for small items, 4 for large ones (two or three, and many rows:
// registers for more warps).
template <int kJoinParts>
__global__ void __launch_bounds__(kJoinRows * 32) cache_attn_join_kernel(const __grid_constant__ CacheAttnArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the partial results are complete from here on
  const int share = blockIdx.x;
  const int4 d = *reinterpret_cast<const int4*>(a.desc + kDescInts * share);
  const int kv_head = a.desc[kDescInts * share + 4];
  if (a.c.status && *reinterpret_cast<volatile int*>(a.c.status) != 0) return;
  const int n_parts = d.x, n_rows = d.y, r0 = d.z;
  if (n_parts <= 0) return;
  for (int r = blockIdx.y * kJoinRows + (threadIdx.x >> 5); r < n_rows; r += kJoinRows * gridDim.y)
    store_joined(a, join_parts<kJoinParts>(a, share, r, n_parts, 0, kJoinParts), r0 + r, d.w, kv_head);
}

// The same for few items in very many parts (a long context on one K/V head: a part per share): block (k, r) looks for the
// k-th item that is in parts, and its 16 warps share the parts of the item's row r.  A warp per row went through 592 parts in
// 37 steps.
constexpr int kWideWarps = 16, kWideParts = 8;
__global__ void __launch_bounds__(kWideWarps * 32, 2) cache_attn_join_wide_kernel(const __grid_constant__ CacheAttnArgs a) {
  __shared__ int n_before[kWideWarps], found;
  __shared__ float m_s[kWideWarps], l_s[kWideWarps];
  __shared__ float4 acc_s[kWideWarps][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the partial results are complete from here on
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) found = -1;
  if (block_stops(a.c)) return;
  int rank = 0;  // items in parts among the shares so far
  for (int s0 = 0; s0 < a.shares; s0 += kWideWarps * 32) {
    const int s = s0 + threadIdx.x;
    const bool here = s < a.shares && a.desc[kDescInts * s] > 0;
    const uint32_t votes = __ballot_sync(0xFFFFFFFFu, here);
    __syncthreads();  // the last round's counts have been read
    if (lane == 0) n_before[warp] = __popc(votes);
    __syncthreads();
    int before = 0;
    for (int w = 0; w < kWideWarps; ++w) {
      before += w < warp ? n_before[w] : 0;
      if (w == warp && here && rank + before + __popc(votes & ((1u << lane) - 1u)) == static_cast<int>(blockIdx.x)) found = s;
    }
    for (int w = 0; w < kWideWarps; ++w) rank += n_before[w];
  }
  __syncthreads();
  const int share = found, r = blockIdx.y;
  if (share < 0) return;
  const int4 d = *reinterpret_cast<const int4*>(a.desc + kDescInts * share);
  if (r >= d.y) return;
  const JoinRow mine = join_parts<kWideParts>(a, share, r, d.x, warp * kWideParts, kWideWarps * kWideParts);
  acc_s[warp][lane] = mine.acc;
  if (lane == 0) {
    m_s[warp] = mine.m;
    l_s[warp] = mine.l;
  }
  __syncthreads();
  if (warp != 0) return;
  JoinRow x{kNoMax, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int w = 0; w < kWideWarps; ++w) x.m = fmaxf(x.m, m_s[w]);
  for (int w = 0; w < kWideWarps; ++w) {
    const float f = ex2_approx(m_s[w] - x.m);
    const float4 v = acc_s[w][lane];
    x.l += l_s[w] * f;
    x.acc.x += v.x * f;
    x.acc.y += v.y * f;
    x.acc.z += v.z * f;
    x.acc.w += v.w * f;
  }
  store_joined(a, x, d.z + r, d.w, a.desc[kDescInts * share + 4]);
}

}  // namespace h3a
