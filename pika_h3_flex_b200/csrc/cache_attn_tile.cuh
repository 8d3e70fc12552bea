// Attention of many new rows over a paged K/V cache: tcgen05 MMAs, the work distribution of cache_attn.cuh.
//
// One CTA per SM walks its share of the units piece by piece.  A piece is up to 2 x 128 query rows (two "streams", each
// floor(128 / group) tokens x the group's heads, so that shared K/V heads fill the rows) against a run of 128-key tiles.
//   warps 0-15       softmax, a warpgroup per stream and 64-key half of every tile, one row per thread (TMEM lane == row)
//   warp 16          producer: TMA loads of Q and of the K and V tiles, page by page, into a ring
//   warps 17, 18     issuers, one per stream: S = Q K^T (N = 64 keys), O += P V (P from TMEM), tcgen05.commit
//   warp 19          cuts the share into pieces and hands them to the others through a small ring: the bookkeeping would
//                    cost every role some 40 registers
//   warps 20-23      helpers, one cache row per thread.  e4m3: widen a staged tile into the ring (below).  bf16: look
//                    at V tiles that not every row sees whole: P is 0 for a key a row does not see, and 0 x NaN is NaN, so
//                    rows behind the last key become zeros and values that are not finite become zeros until they are put
//                    back for the rows that do see them; other tiles go to the MMAs as they are.  And they take the results out of tensor
//                    memory, while the softmax warps are at the next piece.
// TMEM: stream t: S/P buffer of half h at columns [128 t + 64 h, +64), O at [256 + 128 t, +128).  Four chains of S -> P -> O
// run per CTA; the two warpgroups of a stream share the accumulator and so have to agree on each row's reference.
//
// Softmax reference.  Softmax is exact for any reference while the terms stay in range.  A row's is the maximum of its
// logits over the piece's FIRST key tile (the warpgroups exchange it once), which later logits rarely exceed by much: terms
// may grow to 2^60 (bf16 P), 2^14 (fp16 P).  A piece in which some row outgrows that is done again after the others: one
// pass that only looks for the rows' maxima, then one with those as references.  So is one in which terms have grown and large
// values of V took a row's sums out of fp32, as with the maxima for references they would not, and one with logits above 10^6,
// whose products with the scale have to be rounded like their maximum.  Against a running maximum per
// warp, with O rescaled when it moves (two warpgroups, both halves each, two register images of S): that loop was 1.4 K
// instructions and the SM's instruction cache missed on every second request, with helpers and issuers running other code
// beside it (5.5 warps stalled on instruction fetch per issue); the loop here is a quarter of it.
//
// e4m3 tiles become fp16, two instructions per pair: a code is exact in fp16 (one conversion), and so is its product with
// 2^(k - kref), kref being the tile's largest exponent, down to k - kref = -15.  2^kref goes into the tile's softmax scale, and
// Q into fp16 by a power of two per row that joins that scale too.  A K tile whose exponents lie further apart (its largest key
// may weigh nothing, or be hidden, so that all others count with all their bits) keeps the bare codes, and the softmax warps
// multiply each column of S by its key's power first, in tensor memory, so that the ordinary loop stays as short as it is.
// V and O are in units of the largest exponent of the piece's first tile; fp16 holds codes up
// to 2^7 above that, and rows 2^14 below it with all their bits.  A V tile with rows outside that is widened to bf16
// instead, and its P rounded to bf16; one with rows 2^40 above the unit has its piece done again in the largest's units.  (Everything through bf16 took five instructions per pair.)
//
// What bounds it.  A tile of 256 rows x 128 keys is 16.8 MFLOP, 1.5 us of an SM at the rate of the fastest library product;
// it takes 1.9 us (e4m3 2.0): four chains of MMA, 64 exponentials a thread and MMA that wait for one another, under the
// power cap where calls are long.  4,680 rows x 40 heads over 49,384 keys: 3.6 ms by itself, 4.0 ms and 1.16 PFLOP/s among
// other work (e4m3 4.0 ms by itself); 2,048 rows x 40 heads over 20,011 keys of 8 shared heads: 0.61 ms by itself (e4m3 0.70,
// 0.79 among other work).  A piece costs some 3 us beside its tiles (first maxima, last P V, results), which is what is left
// in calls of few tiles each: 6,240 rows x 40 heads over prompts of 512 and 77 tokens 97 us (e4m3 115), 8 new tokens x 32
// heads on each of 32 contexts of 4,000 e4m3 tokens 124 us.
//
// Every wait is bounded: when the limit runs out the CTA raises a CTA-wide flag that the other waits poll, lets copies in
// flight land, records the wait's code in the status word, frees TMEM and returns.  Warps meet at mbarriers, never at named barriers,
// so that one that gave up keeps nobody waiting for ever.
#pragma once
#include "cache_attn.cuh"

namespace h3a {

constexpr int kTileThreads = 768;
constexpr int kKeyTile = 128, kTileKeyShift = 7;
constexpr int kProducerWarp = 16, kIssuerWarp = 17, kPieceWarp = 19, kHelperWarp = 20;
constexpr int kTileRows = 256;         // rows of an item
constexpr int kTileBytes = 32768;      // 128 rows of 128 bf16
constexpr int kTileHalf = 16384;       // one [128 rows][128 bytes] swizzled box
constexpr int kCodeBytes = 16384;      // 128 rows of 128 codes
template <bool kFp8>
struct TileRing {
  static constexpr int kRing = kFp8 ? 3 : 4;     // tiles as the MMAs read them
  static constexpr int kStaged = kFp8 ? 3 : 0;   // e4m3 tiles as loaded
  static constexpr int kBytes = kRing * kTileBytes + kStaged * kCodeBytes;
};

struct TileBars {
  uint64_t full[5];        // ring slot: copies have landed that MMAs may read as they are (bf16)
  uint64_t ready[5];       // ring slot: a helper has written or looked at it
  uint64_t empty[5];       // ring slot: both issuers' MMAs are done with it
  uint64_t staged[4];      // copies have landed that a helper is to look at: e4m3 staging slot; bf16 ring slot
  uint64_t unstaged[4];    // e4m3: widened
  uint64_t q_full[2], q_empty[2];  // [stream]: a phase per piece in which the stream has work, so that nobody has to watch the other's
  uint64_t q_ready[2];     // e4m3: the stream's Q is in fp16
  uint64_t s_full[2][2], p_full[2][2];  // [stream][half]
  uint64_t o_full[2];      // every P V of the stream's piece has completed
  uint64_t o_free[2];      // the helpers have read O
  uint64_t fin[2], fin_free[2];  // the stream's sums and references of a piece are there / have been read
  uint64_t meet[2];        // the stream's eight warps have left what the other half is to see
  uint64_t piece_full[4], piece_empty[4];
  uint64_t tmem_ready;
  uint32_t tmem_base;
  uint32_t early_exit;
  uint32_t more;             // the share has a piece at all
  volatile uint32_t abort_flag;  // code of a wait that gave up: everybody else does too
  uint32_t redo;             // pieces of the current batch that outgrew their reference, a bit each
  float left[2][2][2][128];  // [turn][stream][half][row]: what the halves of a stream leave for each other
  float sums[2][2][128], refs[2][128];  // [stream][half][row], [stream][row]: for the helpers
};
constexpr int kTileBarBytes = 7680;
constexpr int kTileSmemBytes = 2 * kTileBytes + (TileRing<true>::kBytes > TileRing<false>::kBytes ? TileRing<true>::kBytes : TileRing<false>::kBytes) + 1024 + kTileBarBytes;
static_assert(sizeof(TileBars) <= kTileBarBytes, "shared memory layout");
enum : uint32_t {  // status codes of waits that ran out (low byte of the status word)
  kTileWaitEmpty = 33, kTileWaitFull, kTileWaitReady, kTileWaitUnstaged, kTileWaitStaged, kTileWaitQFull, kTileWaitQEmpty,
  kTileWaitQReady, kTileWaitS, kTileWaitP, kTileWaitO, kTileWaitOFree, kTileWaitMeet, kTileWaitPiece, kTileWaitTmem,
  kTileWaitFin, kTileWaitFinFree
};

// There are forty waits, and what a hot loop steps over costs instruction cache too: a wait that gives up only leaves its
// code, which is reported at the end.
struct TileWait {
  const CacheAttnArgs& a;
  TileBars* bars;
  __device__ __forceinline__ static uint32_t now() { return static_cast<uint32_t>(global_timer_ns() >> 10); }
  __device__ __forceinline__ bool one(uint64_t& barrier, uint32_t parity, uint32_t code) const {
    const uint32_t bar = smem_u32(&barrier);
    if (mbar_try_wait(bar, parity)) return true;
    uint32_t polls = 0, t0 = 0;
#pragma unroll 1
    while (!mbar_try_wait(bar, parity)) {
      if ((++polls & 63u) != 0u) continue;
      if (bars->abort_flag) return false;
      if (polls == 64u) t0 = now();
      if (now() - t0 > a.wait_units) {
        bars->abort_flag = code;
        return false;
      }
    }
    return true;
  }
  // the whole warp, with one verdict
  __device__ __forceinline__ bool operator()(uint64_t& barrier, uint32_t parity, uint32_t code) const {
    return __all_sync(0xFFFFFFFFu, one(barrier, parity, code));
  }
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// 32 bytes of one row: a thread owns a row of O, and a warp's store is 32 pieces 256 bytes apart, so that pieces as long as
// a sector count (16 bytes at a time, 256 rows took 5 us, as long as two and a half key tiles).
__device__ __forceinline__ void stg_v8(void* to, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// A piece as the roles see it.
struct TilePiece {
  int n_tiles;       // key tiles [t0, t0 + n_tiles)
  int t0;
  int end[2];        // the stream takes part in the first `end` of them
  int lim_min, lim_max;  // keys that the item's first and last row see
  int b, h;
  int row0;          // packed row of the item's first token
  int tok0, n, len;  // its number in the sequence; new rows and length of the sequence
  int whole;         // the piece is the whole item; otherwise its results are partial
  int tail;          // ... and go to the share's tail slot (the item begins here)
  int mode;          // how the rows' references come about
  int bit;           // its bit in `redo`
  int vref;          // e4m3: O is in units of 2^(vref - 127); left by the producer
  int odd_tile;      // the first tile that not every row sees whole
  volatile int poison;  // left by the helpers: some V row there holds values that counted as zeros ...
  uint32_t odd[12];     // ... a bit per key from that tile on (limits are at most 255 keys apart: three tiles)
};
// e4m3: what a tile's rows were widened with
struct TileInfo {
  int kref;       // the tile's logits are in units of 2^(kref - 127); 0: K as bare codes, each key in units of its own
  int vref;       // V, and so O, is in units of 2^(vref - 127): the same for a piece's tiles
  int wide;       // V is bf16, and P is to be
};
constexpr int kInfoRing = 8;  // the producer is at most four tiles ahead of the softmax warps
// 64 columns of one row of S times `unit`, and times a power of two per key whose exponent bytes are at e_at (0: none).  A
// call of its own: in line, the hot loop around it took 1.5 % longer (chunk of 2,048 over 20,011 keys 806 us against 792).
__device__ __noinline__ void scale_columns(uint32_t s_addr, uint32_t e_at, float unit) {
#pragma unroll 1
  for (int x = 0; x < 64; x += 16) {
    uint32_t r[16];
    uint4 e = make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
    tmem_ld16(s_addr + x, r);
    if (e_at != 0u) ld_shared_v4(e_at + x, e);
    const uint32_t ex[4] = {e.x, e.y, e.z, e.w};
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      asm volatile("" : "+r"(r[i]));  // not before the wait
      const uint32_t power = (ex[i >> 2] >> (8 * (i & 3))) & 0xFFu;
      r[i] = __float_as_uint(__uint_as_float(r[i]) * fminf(unit * __uint_as_float(power << 23), 3.0e38f));
    }
    tmem_st16(s_addr + x, r);
  }
  tmem_wait_st();
}
// whether a row of results, as it was stored (bf16 or fp32), holds a value that is not finite
__device__ __noinline__ bool left_range(const uint8_t* row, bool bf16) {
  bool lost = false;
#pragma unroll 1
  for (int c = 0; c < (bf16 ? 16 : 32); ++c) {
    const uint4 w = *reinterpret_cast<const uint4*>(row + 16 * c);
    const uint32_t top = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
    lost |= bf16 ? non_finite2(top) : top >= 0x7F800000u;
  }
  return lost;
}
// Adds the values of a V row that are not finite to a row of results as it was stored (bf16 or fp32).  Looking for them value
// by value among all keys of the last tiles, a chunk with one NaN in V took 43 times as long as without (bf16, 2,048 tokens x
// 16 heads over 8,192 keys: 5.2 ms against 121 us).
template <bool kFp8>
__device__ __noinline__ void put_back_row(const CacheAttnArgs& a, int b, int h, int key, uint8_t* to, bool bf16) {
  const uint8_t* row = nullptr;
  if constexpr (!kFp8) {
    const int slot = a.c.by_page(key);
    row = a.c.pool[1] + checked_page(a, b, slot) * a.c.page_bytes[1] + (key - slot * a.c.page_size) * a.c.token_bytes[1] + h * a.c.head_bytes[1];
  }
#pragma unroll 1
  for (int d0 = 0; d0 < kCacheDim; d0 += 2) {
    const uint32_t w = kFp8 ? 0x7FFF7FFFu : __ldg(reinterpret_cast<const uint32_t*>(row + 2 * d0));  // a row of codes is NaN as a whole
    if (!non_finite2(w)) continue;
    for (int x = 0; x < 2; ++x) {
      const float v = __uint_as_float(x ? w & 0xFFFF0000u : w << 16);
      if (isfinite(v)) continue;
      if (bf16) {
        __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(to) + d0 + x;
        *o = static_cast<__nv_bfloat16>(static_cast<float>(*o) + v);
      } else {
        reinterpret_cast<float*>(to)[d0 + x] += v;
      }
    }
  }
}
// 2^-d as an fp16 pair, d >= -15
__device__ __forceinline__ uint32_t f16x2_pow2_neg(int d) {
  const uint32_t h = d <= 14 ? static_cast<uint32_t>(15 - d) << 10 : d <= 24 ? 1u << (24 - d) : 0u;
  return h * 0x10001u;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A row of 128 codes (at `src`, 16-byte pieces swizzled by the row like the copies that brought them) as 128 bf16 or fp16
// values times `f` (bf16: and times `f2`, what of a
// power of two the type's largest exponent leaves over), in the two half boxes at `dst`.  The pieces are read four at a time: one by one, a piece waited for the
// one before it, and the helpers for them all (1,100 cycles for 16 KB).
template <bool kBf16>
__device__ __forceinline__ void widen_row(uint32_t src, uint32_t dst, uint32_t swz, uint32_t f, uint32_t f2, bool blank) {
#pragma unroll 1
  for (int c0 = 0; c0 < 8; c0 += 4) {
    uint4 w[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) ld_shared_v4(src + (((c0 + c) ^ swz) << 4), w[c]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t in[4] = {blank ? 0u : w[c].x, blank ? 0u : w[c].y, blank ? 0u : w[c].z, blank ? 0u : w[c].w};
      uint32_t o[8];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if constexpr (kBf16) {
          o[2 * y] = mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(in[y], 0, 0x1404)), f), f2);
          o[2 * y + 1] = mul_bf16x2(mul_bf16x2(e4m3_pattern(__byte_perm(in[y], 0, 0x3424)), f), f2);
        } else {
          o[2 * y] = mul_f16x2(e4m3_to_f16x2(in[y]), f);
          o[2 * y + 1] = mul_f16x2(e4m3_high_to_f16x2(in[y]), f);
        }
      }
      const uint32_t at = dst + (c0 >> 2) * kTileHalf;
      st_shared_v4(at + (((2 * c) ^ swz) << 4), o[0], o[1], o[2], o[3]);
      st_shared_v4(at + (((2 * c + 1) ^ swz) << 4), o[4], o[5], o[6], o[7]);
    }
  }
}
constexpr int kPieceRing = 4;
constexpr int kPieceReaders = 23;  // warps
constexpr int kPieceBatch = 32;    // pieces between two looks at `redo`
enum : int { kFirstTile = 0, kFindMaxima = 1, kUseMaxima = 2 };

__device__ __forceinline__ int piece_limit(const CacheAttnArgs& a, const TilePiece& q, int token) {
  return a.causal ? max(0, min(q.len, q.len - q.n + token + 1)) : q.len;
}
__device__ __forceinline__ void describe_piece(const CacheAttnArgs& a, const ShareIter& iter, const Piece& p, TilePiece& q) {
  const int T = a.item_tokens >> 1;
  q.tok0 = p.it * a.item_tokens;
  q.n_tiles = p.t1 - p.t0;
  q.t0 = p.t0;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = q.tok0 + t * T, last = min(p.s.n, first + T) - 1;
    q.end[t] = last >= first ? max(0, min(p.t1, (key_limit(a, p.s, last) + kKeyTile - 1) / kKeyTile) - p.t0) : 0;
  }
  q.lim_min = key_limit(a, p.s, q.tok0);
  q.lim_max = key_limit(a, p.s, item_last_token(a, p.s, p.it));
  q.odd_tile = max(p.t0, q.lim_min >> kTileKeyShift);
  q.poison = 0;
  q.b = p.b;
  q.h = p.h;
  q.row0 = p.s.s0 + q.tok0;
  q.n = p.s.n;
  q.len = p.s.len;
  q.whole = p.first && p.last;
  q.tail = p.first;
  if (p.first && !p.last) {
    const int r0 = q.tok0 * a.group;
    describe_join(a, iter, iter.item_base + a.set_up + item_tiles(a, p.s, p.it), min(p.s.n * a.group - r0, a.item_tokens * a.group), r0, p.s.s0, p.h);
  }
}

// The same value in every lane, in a form that lets the compiler know it: what is computed from it, descriptors of MMAs
// above all, then lives in uniform registers (moved there from ordinary ones before each, an MMA took 90 cycles to issue).
__device__ __forceinline__ int uniform(int x) { return __reduce_max_sync(0xFFFFFFFFu, x); }

// rows [0, box_rows) of a 4-D page box are whole keys of one page: box_rows divides the page size and the tile
template <bool kFp8>
__global__ void __launch_bounds__(kTileThreads, 1)
cache_attn_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const int box_rows, const __grid_constant__ CacheAttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ ShareStart start;
  __shared__ TilePiece pieces[kPieceRing];  // n_tiles < 0: no more
  __shared__ ShareIter walk, again;         // the piece warp's: where it is in the share, where its batch began
  __shared__ Piece p;
  __shared__ TileInfo info[kInfoRing];
  __shared__ alignas(16) uint8_t exps[kInfoRing][2][kKeyTile];  // e4m3: the exponent bytes of a tile's rows of K and V
  static_assert(kTileSmemBytes + sizeof(ShareStart) + sizeof(TilePiece) * kPieceRing + 2 * sizeof(ShareIter) + sizeof(Piece) + (sizeof(TileInfo) + 2 * kKeyTile) * kInfoRing <= 232448, "shared memory budget");
  using R = TileRing<kFp8>;
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);
  const uint32_t q_smem = base, ring = base + 2 * kTileBytes, staging = ring + R::kRing * kTileBytes;
  TileBars* bars = reinterpret_cast<TileBars*>(smem + kTileSmemBytes - 1024 - kTileBarBytes);
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < R::kRing; ++i) {
      mbar_init(smem_u32(&bars->full[i]), 1);
      mbar_init(smem_u32(&bars->ready[i]), 4);   // one arrive per helper warp
      mbar_init(smem_u32(&bars->empty[i]), 2);   // one commit per issuer
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&bars->staged[i]), 1);
      mbar_init(smem_u32(&bars->unstaged[i]), 4);
    }
    mbar_init(smem_u32(&bars->tmem_ready), 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&bars->q_full[t]), 1);
      mbar_init(smem_u32(&bars->q_empty[t]), 1);
      mbar_init(smem_u32(&bars->q_ready[t]), 8);
      for (int hf = 0; hf < 2; ++hf) {
        mbar_init(smem_u32(&bars->s_full[t][hf]), 1);
        mbar_init(smem_u32(&bars->p_full[t][hf]), 4);
      }
      mbar_init(smem_u32(&bars->o_full[t]), 1);
      mbar_init(smem_u32(&bars->o_free[t]), 4);
      mbar_init(smem_u32(&bars->fin[t]), 8);
      mbar_init(smem_u32(&bars->fin_free[t]), 4);
      mbar_init(smem_u32(&bars->meet[t]), 8);
    }
    for (int i = 0; i < kPieceRing; ++i) {
      mbar_init(smem_u32(&bars->piece_full[i]), 1);
      mbar_init(smem_u32(&bars->piece_empty[i]), kPieceReaders);
    }
    bars->abort_flag = 0;
    bars->redo = 0;
    bars->early_exit = (a.c.status != nullptr && *reinterpret_cast<volatile int*>(a.c.status) != 0) ? 1u : 0u;
    fence_mbar_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  allow_next_launch();
  {
    ShareIter begin = share_begin(a, &start);
    if (threadIdx.x == kPieceWarp * 32) {  // the first piece is found here, in registers: everybody waits for it
      a.desc[kDescInts * blockIdx.x] = 0;  // by the thread that may go on to describe an item there: no other order is needed
      again = begin;
      bars->more = begin.next(a, p);
      if (bars->more) describe_piece(a, begin, p, pieces[0]);
      walk = begin;
    }
  }
  __syncthreads();  // barriers and flags are set up
  if (bars->early_exit) return;
  const TileWait wait{a, bars};
  const int T = a.item_tokens >> 1;
  // the readers' side of the ring of pieces
  uint32_t n_pieces = 0;
  auto piece = [&]() -> const TilePiece* {
    const uint32_t i = n_pieces % kPieceRing;
    if (!wait(bars->piece_full[i], (n_pieces / kPieceRing) & 1, kTileWaitPiece) || pieces[i].n_tiles < 0) return nullptr;
    return &pieces[i];
  };
  auto piece_done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bars->piece_empty[n_pieces % kPieceRing]));
    ++n_pieces;
  };

  // Tensor memory is allocated by the first issuer while the first tiles are on their way; who uses it waits for that.
  auto tensor_memory = [&](bool& ok) -> uint32_t {
    ok = wait(bars->tmem_ready, 0, kTileWaitTmem);
    tc_fence_after_sync();
    return static_cast<uint32_t>(uniform(static_cast<int>(bars->tmem_base)));
  };

  if (warp >= kHelperWarp) {
    // =========================================================== helpers: thread r owns row r of every tile
    const int row = threadIdx.x - kHelperWarp * 32;
    const uint32_t swz = row & 7;
    int cnt = 0;
    uint32_t n_done = 0;   // tiles so far, all pieces
    uint32_t n_out = 0;    // pieces whose results have left: the phase of fin
    uint32_t o_phase = 0;  // bit t: the phase of o_full[t]
    uint32_t v_phase = 0;  // bf16: bit s: the phase of staged[s]
    bool ok = true;
    // which rows of a V tile counted as zeros, for the epilogue
    auto leave_odd = [&](const TilePiece* q, int tile, bool odd) {
      const uint32_t votes = __ballot_sync(0xFFFFFFFFu, odd);
      if (lane == 0) {
        TilePiece* to = const_cast<TilePiece*>(q);
        to->odd[4 * (tile - to->odd_tile) + (warp & 3)] = votes;
        if (votes != 0u) to->poison = 1;
      }
    };
    const TilePiece* held = nullptr;  // a piece whose results are still in tensor memory
#pragma unroll 1
    for (;;) {
      // The next piece's first K goes ahead of this one's results, its V between the two streams', but nobody waits for a
      // piece before results have left.
      const TilePiece* q = nullptr;
      bool last = false;
      if (held == nullptr || __all_sync(0xFFFFFFFFu, mbar_test_wait(smem_u32(&bars->piece_full[n_pieces % kPieceRing]), (n_pieces / kPieceRing) & 1))) {
        q = piece();
        last = q == nullptr;
      }
      const int n_tiles = q ? uniform(q->n_tiles) : 0, t0 = q ? uniform(q->t0) : 0;
      const int lim_min = q ? uniform(q->lim_min) : 0, lim_max = q ? uniform(q->lim_max) : 0;
      const int steps = max(2 * n_tiles, held ? 2 : 0);
#pragma unroll 1
      for (int step = 0; ok && step < steps; ++step) {
        const int x = step & 1, tile = t0 + (step >> 1), key = tile * kKeyTile + row;  // K, then V
        const bool special = (tile + 1) * kKeyTile > lim_min;
        const bool gone = key >= lim_max;
        if (step < 2 * n_tiles && (kFp8 || (x == 1 && special))) {
          const int s = cnt % R::kRing;
          const uint32_t dst = ring + s * kTileBytes + row * 128;
          if constexpr (kFp8) {
            const int g = cnt % R::kStaged;
            ok = wait(bars->staged[g], (cnt / R::kStaged) & 1, kTileWaitStaged) && wait(bars->empty[s], ((cnt / R::kRing) & 1) ^ 1, kTileWaitEmpty);
            if (!ok) break;
            const uint32_t src = staging + g * kCodeBytes + row * 128;
            // what the producer has found out about the tile; a row that is not there may hold anything, codes for NaN
            // included, and counts as zeros, as does for now a row that is not finite and that not every query row sees
            const TileInfo in = info[n_done % kInfoRing];
            const int e = exps[n_done % kInfoRing][x][row];
            const bool put_back = x == 1 && special && !gone && e == 255;
            if (x == 1 && special) leave_odd(q, tile, put_back);
            const bool none = gone || put_back;
            const int d = x ? in.vref - e : in.kref != 0 ? in.kref - e : 0;  // the row's power of two against the unit's
            if (x == 1 && in.wide) {
              // 2^(120 - d) in two steps: a row may be 2^40 above the unit (beyond that the piece is done again)
              const uint32_t f = none ? 0u : e == 255 ? 0x7FFF7FFFu : static_cast<uint32_t>(max(0, min(254, 247 - d))) * 0x800080u;
              widen_row<true>(src, dst, swz, f, static_cast<uint32_t>(max(127, min(254, 120 - d))) * 0x800080u, none);
            } else {
              widen_row<false>(src, dst, swz, none ? 0u : e == 255 ? 0x7FFF7FFFu : f16x2_pow2_neg(d), 0, none);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(smem_u32(&bars->ready[s]));
              mbar_arrive(smem_u32(&bars->unstaged[g]));
            }
          } else {
            ok = wait(bars->staged[s], (v_phase >> s) & 1, kTileWaitStaged);
            if (!ok) break;
            v_phase ^= 1u << s;
            uint32_t m = 0;  // the row's largest magnitude by its bits
#pragma unroll 4
            for (int c = 0; c < 16; ++c) {
              const uint32_t at = dst + (c >> 3) * kTileHalf + (((c & 7) ^ swz) << 4);
              uint4 w = make_uint4(0, 0, 0, 0);
              if (gone) st_shared_v4(at, 0, 0, 0, 0);
              else ld_shared_v4(at, w);
              m = __vmaxu2(m, __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu)));
            }
            leave_odd(q, tile, non_finite2(m));
            if (non_finite2(m)) {  // rare
#pragma unroll 1
              for (int c = 0; c < 16; ++c) {
                const uint32_t at = dst + (c >> 3) * kTileHalf + (((c & 7) ^ swz) << 4);
                uint4 w;
                ld_shared_v4(at, w);
                st_shared_v4(at, finite_or_zero2(w.x), finite_or_zero2(w.y), finite_or_zero2(w.z), finite_or_zero2(w.w));
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars->ready[s]));
          }
        }
        if (step < 2 * n_tiles) {
          ++cnt;
          n_done += x;
        }
        if (step > 1 || !held) continue;
        // ---- results of the piece before, a stream: thread r has row r
        const int t = step;
        const uint32_t tmem = tensor_memory(ok);
        const bool whole = held->whole != 0, keep = held->mode != kFindMaxima;
        const bool any = uniform(held->end[t]) > 0;
        ok = ok && wait(bars->fin[t], n_out & 1, kTileWaitFin) && (!any || wait(bars->o_full[t], (o_phase >> t) & 1, kTileWaitO));
        if (!ok) break;
        if (any) o_phase ^= 1u << t;
        tc_fence_after_sync();
        const float l_sum = bars->sums[t][0][row] + bars->sums[t][1][row], m_ref = bars->refs[t][row];
        const int row_i = a.by_group(row), row_token = t * T + row_i;  // row r: token r / group, head r % group
        const bool have_row = keep && row < T * a.group && held->tok0 + row_token < held->n;
        const int head = held->h * a.group + row - row_i * a.group;
        const long long out_row = held->row0 + row_token;
        const float unit = kFp8 ? __uint_as_float(static_cast<uint32_t>(any ? held->vref : 0) << 23) : 1.0f;
        const float f = whole ? (l_sum == 0.f ? 0.f : 1.0f / l_sum) * unit : unit;
        uint8_t* dst;
        if (whole) {
          dst = reinterpret_cast<uint8_t*>(a.o + out_row * a.o_stride_l + head * a.o_stride_h);
          if (have_row && a.lse)
            a.lse[static_cast<long long>(head) * a.c.rows + out_row] = l_sum == 0.f ? -INFINITY : (m_ref + log2f(l_sum)) * 0.6931471805599453f;
        } else {
          float* part = part_slot(a, blockIdx.x, held->tail != 0) + t * T * a.group * kCacheDim;
          dst = reinterpret_cast<uint8_t*>(part + row * kCacheDim);
          if (have_row) {
            float* stat = part_slot(a, blockIdx.x, held->tail != 0) + kTileRows * kCacheDim + t * T * a.group + row;
            stat[0] = m_ref;
            stat[kTileRows] = l_sum;
          }
        }
        const uint32_t from = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + 256 + t * 128;
        uint32_t s[16] = {};
        if (any) tmem_ld16(from, s);
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {  // 16 dims at a time, the next 16 on their way while these are stored
          float o[16];
          if (any) {
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(s[i]));
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __uint_as_float(s[i]) * f;
          if (c < 7) {
            if (any) tmem_ld16(from + 16 * (c + 1), s);
          } else {  // the next piece may have O and the sums
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              if (any) mbar_arrive(smem_u32(&bars->o_free[t]));
              mbar_arrive(smem_u32(&bars->fin_free[t]));
            }
          }
          if (!have_row) continue;
          if (whole) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(o[2 * i], o[2 * i + 1]);
            if (a.o_sectors) {
              stg_v8(dst + 32 * c, w);
            } else {
              *reinterpret_cast<uint4*>(dst + 32 * c) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(dst + 32 * c + 16) = make_uint4(w[4], w[5], w[6], w[7]);
            }
          } else {
            stg_v8(dst + 64 * c, reinterpret_cast<const uint32_t*>(o));
            stg_v8(dst + 64 * c + 32, reinterpret_cast<const uint32_t*>(o + 8));
          }
        }
        // rare: terms have grown (the sum is larger than one of so many terms up to the reference's own) and a sum has left fp32
        if (l_sum > (kFp8 ? 4.f : 1.f) * kKeyTile * held->n_tiles && have_row && held->mode == kFirstTile) {
          if (left_range(dst, whole)) atomicOr(&bars->redo, 1u << held->bit);
        }
        if (held->poison != 0 && have_row) {  // rare: values left out above are added to the stored row, if it sees them
          const int end = min(piece_limit(a, *held, held->tok0 + row_token), (held->t0 + held->n_tiles) * kKeyTile);
          int key0 = held->odd_tile * kKeyTile;
          for (int w = 0; key0 < end; ++w, key0 += 32)
            for (uint32_t bits = held->odd[w]; bits != 0u; bits &= bits - 1u) {
              const int key = key0 + __ffs(bits) - 1;
              if (key < end) put_back_row<kFp8>(a, held->b, held->h, key, dst, whole);
            }
        }
        if (t == 1) {
          ++n_out;
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bars->piece_empty[(n_pieces - 1) % kPieceRing]));
          held = nullptr;
        }
      }
      if (!ok || last) break;
      if (q) {
        held = q;
        ++n_pieces;
      }
    }
  } else if (warp >= kProducerWarp) {
    if (warp == kProducerWarp) {
      // ========================================================= producer: lane x copies sub-box x of a tile
      const int n_boxes = kKeyTile / box_rows;
      const int box_bytes = box_rows * (kFp8 ? kCacheDim : 2 * kCacheDim);
      const uint32_t q_bytes = T * a.group * 256;
      int cnt = 0;
      uint32_t n_done = 0;  // tiles so far, all pieces
      int vref = 0;         // e4m3: V's unit in the piece
      uint32_t q_phase = 3;  // bit t: the phase of q_empty[t], whose first wait is for nothing
      bool ok = true;
      const TilePiece* q;
#pragma unroll 1
      for (; ok && (q = piece()) != nullptr; piece_done()) {
        const int n_tiles = uniform(q->n_tiles), t0 = uniform(q->t0), b = uniform(q->b), h = uniform(q->h), lim_max = uniform(q->lim_max);
        const int mode = uniform(q->mode), lim_min = uniform(q->lim_min);
        if (n_tiles == 0) continue;
        const int n_streams = uniform((q->end[0] > 0 ? 1 : 0) | (q->end[1] > 0 ? 2 : 0));
        // Q is free late in the previous piece, ring slots earlier: the first K tile goes ahead of Q, but for the first piece,
        // where it has to wait for page numbers
        auto load_q = [&]() {
#pragma unroll 1
          for (int t = 0; ok && t < 2; ++t) {
            if (((n_streams >> t) & 1) == 0) continue;
            ok = wait(bars->q_empty[t], (q_phase >> t) & 1, kTileWaitQEmpty);
            if (!ok) break;
            q_phase ^= 1u << t;
            const uint32_t bar = smem_u32(&bars->q_full[t]);
            if (lane == 0) mbar_arrive_expect_tx(bar, q_bytes);
            __syncwarp();
            if (lane < 2) tma_load_3d(q_smem + t * kTileBytes + lane * kTileHalf, &tm_q, bar, 64 * lane, h * a.group, q->row0 + t * T);
            __syncwarp();
          }
        };
        if (n_pieces == 0) load_q();
        // A lane looks after 4 rows of every tile, which are in one page.  Its page number is fetched two tiles ahead, the rows'
        // exponent bytes (e4m3) one tile ahead; nothing looks at either before it is needed, or the loads would be waited for.
        int id = 0, id_next = 0;
        uint32_t raw_k[4] = {}, raw_v[4] = {};
        auto fetch_id = [&](int tile) {
          const int key = tile * kKeyTile + lane * 4;
          return key < lim_max ? __ldg(a.c.pages + b * a.c.pages_stride + a.c.by_page(key)) : 0;
        };
        auto checked = [&](int raw) {  // a page that does not exist is reported, and some other page read
          if (static_cast<unsigned>(raw) < static_cast<unsigned>(a.c.n_pages)) return raw;
          report_cache(a.c, b);
          return 0;
        };
        auto fetch_ex = [&](int tile, int page) {
          const int key = tile * kKeyTile + lane * 4, at = key - a.c.by_page(key) * a.c.page_size;
          const uint8_t* from_k = a.c.exps[0] + page * a.c.exp_page[0] + at * a.c.exp_token[0] + h * a.c.exp_head[0];
          const uint8_t* from_v = a.c.exps[1] + page * a.c.exp_page[1] + at * a.c.exp_token[1] + h * a.c.exp_head[1];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            raw_k[i] = key + i < lim_max ? __ldg(from_k + i * a.c.exp_token[0]) : 0u;
            raw_v[i] = key + i < lim_max ? __ldg(from_v + i * a.c.exp_token[1]) : 0u;
          }
        };
        id_next = fetch_id(t0);
        int v_most = 0;                       // largest exponent of V in the piece
        if (mode != kUseMaxima) vref = 0;     // otherwise what the pass before found
#pragma unroll 1
        for (int it = -1; ok && it < n_tiles; ++it) {
          const int tile = t0 + it;
          // sub-box x of the tile: lane x copies it; none behind the last key
          const int key = tile * kKeyTile + lane * box_rows, at = key - a.c.by_page(key) * a.c.page_size;
          const bool mine = lane < n_boxes && key < lim_max;
          const uint32_t bytes = __popc(__ballot_sync(0xFFFFFFFFu, mine)) * box_bytes;
          const int page = __shfl_sync(0xFFFFFFFFu, id, (lane * box_rows / 4) & 31);
          if (kFp8 && it >= 0) {
            // the tile's largest and smallest exponents, rows that are not finite (255) aside, and of V rows of nothing (7) too
            uint32_t k_top = 0, k_low = 255, v_top = 0, v_low = 255;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t x = raw_k[i], y = raw_v[i];
              if (x != 255u) k_top = max(k_top, x);
              if (x != 0u) k_low = min(k_low, x);  // 0: no key
              if (y > 7u && y != 255u) {
                v_top = max(v_top, y);
                v_low = min(v_low, y);
              }
            }
            k_top = __reduce_max_sync(0xFFFFFFFFu, k_top);
            k_low = __reduce_min_sync(0xFFFFFFFFu, k_low);
            v_top = __reduce_max_sync(0xFFFFFFFFu, v_top);
            v_low = __reduce_min_sync(0xFFFFFFFFu, v_low);
            const int vt = static_cast<int>(v_top), vl = static_cast<int>(v_low);
            v_most = max(v_most, vt);
            if (vref == 0) vref = vt != 0 ? vt : 127;
            const uint32_t slot = n_done % kInfoRing;
            *reinterpret_cast<uint32_t*>(&exps[slot][0][4 * lane]) = raw_k[0] | (raw_k[1] << 8) | (raw_k[2] << 16) | (raw_k[3] << 24);
            *reinterpret_cast<uint32_t*>(&exps[slot][1][4 * lane]) = raw_v[0] | (raw_v[1] << 8) | (raw_v[2] << 16) | (raw_v[3] << 24);
            if (lane == 0) {
              info[slot].kref = k_top > k_low + 15u ? 0 : static_cast<int>(k_top);
              info[slot].vref = vref;
              if (it == 0) const_cast<TilePiece*>(q)->vref = vref;
              info[slot].wide = vl + 14 < vref || vt > vref + 7;
              // O itself could leave fp32 (the first tile's V next to nothing): with the piece's largest exponent as the unit it cannot
              if (vt > vref + 40) atomicOr(&bars->redo, 1u << q->bit);
            }
          }
          id = checked(id_next);
          id_next = fetch_id(tile + 2);
          if constexpr (kFp8) fetch_ex(tile + 1, id);
          if (it < 0) continue;  // only the fetches
#pragma unroll 1
          for (int x = 0; ok && x < 2; ++x, ++cnt) {
            if (it == 0 && x == 1 && n_pieces > 0) load_q();
            if (!ok) break;
            const CUtensorMap* tm = x ? &tm_v : &tm_k;
            uint32_t dst, bar;
            if constexpr (kFp8) {
              const int s = cnt % R::kStaged;
              ok = wait(bars->unstaged[s], ((cnt / R::kStaged) & 1) ^ 1u, kTileWaitUnstaged);
              dst = staging + s * kCodeBytes + lane * box_rows * 128;
              bar = smem_u32(&bars->staged[s]);
            } else {
              const int s = cnt % R::kRing;
              ok = wait(bars->empty[s], ((cnt / R::kRing) & 1) ^ 1u, kTileWaitEmpty);
              dst = ring + s * kTileBytes + lane * box_rows * 128;
              bar = smem_u32(x == 1 && (tile + 1) * kKeyTile > lim_min ? &bars->staged[s] : &bars->full[s]);
            }
            if (!ok) break;
            __syncwarp();  // with what was left about the tile
            if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
            __syncwarp();
            if (mine) {
              tma_load_4d(dst, tm, bar, 0, at, h, page);
              if constexpr (!kFp8) tma_load_4d(dst + kTileHalf, tm, bar, 64, at, h, page);
            }
            __syncwarp();
          }
          ++n_done;
        }
        if (mode == kFindMaxima) vref = v_most != 0 ? v_most : 127;
      }
    } else if (warp < kPieceWarp) {
      // ========================================================= issuers, one warp per stream
      const int t = warp - kIssuerWarp;
      const uint32_t leader = elect_one();
      constexpr uint32_t kFmt = kFp8 ? UMMA_FMT_F16 : UMMA_FMT_BF16;
      constexpr uint32_t idesc_s = umma_idesc(kFmt, kFmt, 0, 0, 128, 64);
      constexpr uint32_t idesc_pv = umma_idesc(kFmt, kFmt, 0, 1, 128, 128), idesc_pv_wide = umma_idesc(UMMA_FMT_BF16, UMMA_FMT_BF16, 0, 1, 128, 128);
      const uint64_t q_desc = umma_desc_sw128(q_smem + t * kTileBytes, 16, 1024);
      const uint64_t k_desc0 = umma_desc_sw128(ring, 16, 1024);
      const uint64_t v_desc0 = umma_desc_sw128(ring, kTileHalf, 1024);
      if (t == 0) {
        tmem_alloc(smem_u32(&bars->tmem_base), 512);
        tmem_relinquish();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars->tmem_ready));
      }
      bool ok = true;
      const uint32_t tmem = tensor_memory(ok);
      const uint32_t s_tmem = tmem + t * 128, o_tmem = tmem + 256 + t * 128;
      uint32_t p_cnt[2] = {0, 0};  // P halves consumed so far: the phase of p_full
      uint32_t pv_cnt = 0;         // P V groups of the current piece: the first one overwrites O
      uint32_t own = 0;            // pieces in which this stream had work: the phase of q_full, q_ready and o_free
      int c0 = 0;                  // ring tiles before the current piece
      auto issue_s = [&](int hf, int s) {
        const uint64_t kd = k_desc0 + static_cast<uint64_t>((s * kTileBytes + hf * 8192) >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t off = ((k >> 2) * kTileHalf + (k & 3) * 32) >> 4;
          umma_bf16_ss_if(leader, s_tmem + hf * 64, q_desc + off, kd + off, idesc_s, k > 0);
        }
        umma_commit_if(leader, smem_u32(&bars->s_full[t][hf]));
      };
      auto issue_pv = [&](int hf, int s, uint32_t idesc) {
        const uint64_t vd = v_desc0 + static_cast<uint64_t>((s * kTileBytes + hf * 8192) >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_bf16_ts_if(leader, o_tmem, s_tmem + hf * 64 + k * 8, vd + (k * 2048 >> 4), idesc, (pv_cnt > 0 || k > 0) ? 1u : 0u);
        ++pv_cnt;
      };
      // bf16 tiles are read as the copies leave them, but for V tiles that a helper has to look at (which have barriers of
      // their own: nobody has to watch a phase that is not his)
      uint32_t full_phase = 0, ready_phase = 0;  // bit s: the phase of full[s], ready[s]
      auto ready = [&](int c, bool looked_at) {
        const int s = c % R::kRing;
        bool got;
        if (kFp8 || looked_at) {
          got = wait(bars->ready[s], (ready_phase >> s) & 1, kTileWaitReady);
          ready_phase ^= 1u << s;
        } else {
          got = wait(bars->full[s], (full_phase >> s) & 1, kTileWaitFull);
          full_phase ^= 1u << s;
        }
        tc_fence_after_sync();
        return got;
      };
      const TilePiece* q;
#pragma unroll 1
      for (; ok && (q = piece()) != nullptr; piece_done()) {
        const int n_tiles = uniform(q->n_tiles), n_mine = uniform(q->end[t]), t0 = uniform(q->t0), lim_min = uniform(q->lim_min);
        if (n_tiles == 0) continue;
        if (n_mine > 0) ok = wait(kFp8 ? bars->q_ready[t] : bars->q_full[t], own & 1, kFp8 ? kTileWaitQReady : kTileWaitQFull);
        ok = ok && ready(c0, false);
        if (!ok) break;
        pv_cnt = 0;
        if (n_mine > 0) {
          issue_s(0, c0 % R::kRing);
          issue_s(1, c0 % R::kRing);
        }
        umma_commit_if(leader, smem_u32(&bars->empty[c0 % R::kRing]));
#pragma unroll 1
        for (int it = 0; ok && it < n_tiles; ++it) {
          const bool has_next = it + 1 < n_tiles;
          const int cv = c0 + 2 * it + 1, ck = cv + 1;
          if (it + 1 == n_mine) umma_commit_if(leader, smem_u32(&bars->q_empty[t]));  // every S MMA of the stream's piece has been issued
          ok = ready(cv, (t0 + it + 1) * kKeyTile > lim_min);
          if (!ok) break;
          bool k_ready = false;
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            if (ok && it < n_mine) {
              ok = wait(bars->p_full[t][hf], p_cnt[hf] & 1, kTileWaitP);
              // the helpers have read the previous piece's O
              if (ok && pv_cnt == 0 && own > 0) ok = wait(bars->o_free[t], (own - 1) & 1, kTileWaitOFree);
              if (ok) {
                ++p_cnt[hf];
                tc_fence_after_sync();
                issue_pv(hf, cv % R::kRing, kFp8 && info[((c0 >> 1) + it) % kInfoRing].wide ? idesc_pv_wide : idesc_pv);
              }
            }
            if (ok && has_next && !k_ready) {
              ok = ready(ck, false);
              k_ready = ok;
            }
            if (ok && has_next && it + 1 < n_mine) issue_s(hf, ck % R::kRing);
          }
          if (!ok) break;
          umma_commit_if(leader, smem_u32(&bars->empty[cv % R::kRing]));
          if (has_next) umma_commit_if(leader, smem_u32(&bars->empty[ck % R::kRing]));
        }
        if (!ok) break;
        c0 += 2 * n_tiles;
        if (n_mine > 0) {
          umma_commit_if(leader, smem_u32(&bars->o_full[t]));
          ++own;
        }
      }
    } else if (lane == 0) {
      // ========================================================= the share's pieces, one after the other
      uint32_t n = 0;  // pieces handed out
      bool ok = true;
      auto all_done = [&]() {  // everybody has finished every piece handed out
        for (uint32_t k = n < kPieceRing ? 0 : n - kPieceRing; ok && k < n; ++k)
          ok = wait.one(bars->piece_empty[k % kPieceRing], (k / kPieceRing) & 1, kTileWaitPiece);
      };
      bool more = bars->more != 0u, redoing = false, second = false;
      int in_batch = 0, k = 0;  // pieces of the batch; the one that is looked at again
      uint32_t redo = 0;
      if (more) {  // the first piece has been described already
        pieces[0].mode = kFirstTile;
        pieces[0].bit = in_batch++;
        mbar_arrive(smem_u32(&bars->piece_full[0]));
        n = 1;
      }
#pragma unroll 1
      while (ok && (more || redoing)) {
        ShareIter& from = redoing ? again : walk;
        int mode = kFirstTile, bit = 31;
        if (second) {
          second = false;
          mode = kUseMaxima;
        } else if ((redoing ? k : in_batch) < (redoing ? in_batch : kPieceBatch) && from.next(a, p)) {
          if (redoing) {
            if (((redo >> k++) & 1u) == 0u) continue;
            second = true;
            mode = kFindMaxima;
          } else {
            bit = in_batch++;
          }
        } else {  // the batch, or what of it was to be done again, has been handed out
          all_done();
          if (!redoing) more = in_batch == kPieceBatch;
          redo = redoing ? 0u : bars->redo;
          bars->redo = 0;
          redoing = redo != 0u;
          k = 0;
          if (!redoing) {
            again = walk;
            in_batch = 0;
          }
          continue;
        }
        const uint32_t i = n % kPieceRing;
        ok = wait.one(bars->piece_empty[i], ((n / kPieceRing) & 1) ^ 1u, kTileWaitPiece);
        if (!ok) break;
        describe_piece(a, from, p, pieces[i]);
        pieces[i].mode = mode;
        pieces[i].bit = bit;
        mbar_arrive(smem_u32(&bars->piece_full[i]));
        ++n;
      }
      if (ok) {
        const uint32_t i = n % kPieceRing;
        if (wait.one(bars->piece_empty[i], ((n / kPieceRing) & 1) ^ 1u, kTileWaitPiece)) {
          pieces[i].n_tiles = -1;
          mbar_arrive(smem_u32(&bars->piece_full[i]));
        }
      }
    }
    __syncwarp();
  } else {
    // =========================================================== softmax and results
    const int t = (warp >> 2) & 1, hf = warp >> 3, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    bool ok = true;
    const uint32_t tmem = tensor_memory(ok);
    const uint32_t s_addr = tmem + lane_base + t * 128 + hf * 64;
    constexpr float kLift = kFp8 ? 2.f : 0.f;            // the reference's own term is 2^kLift
    constexpr float kMostTerms = kFp8 ? 6.0e4f : 1.0e18f;  // 64 terms of a row: more than that has outgrown the reference
    uint32_t j = 0;         // key tiles the stream has processed: the phase of s_full
    uint32_t own = 0;       // pieces in which the stream had work: the phase of q_full
    uint32_t n_fin = 0;     // pieces so far: the phase of fin_free
    uint32_t n_before = 0;  // tiles of the pieces before
    uint32_t turn = 0;      // meetings of the stream's two halves so far
    // Leaves x for the same row's thread of the other half and returns what that one left.  Each side's values are in a
    // slot by turn: nobody can be two meetings ahead of a reader.
    auto exchange = [&](float x) -> float {
      bars->left[turn & 1][t][hf][row] = x;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars->meet[t]));
      ok = wait(bars->meet[t], turn & 1, kTileWaitMeet);
      const float y = bars->left[turn & 1][t][hf ^ 1][row];
      ++turn;
      return y;
    };
    const TilePiece* q;
#pragma unroll 1
    for (; ok && (q = piece()) != nullptr; piece_done()) {
      const int n_mine = uniform(q->end[t]), mode = uniform(q->mode);
      const int row_i = a.by_group(row);                  // row r: token r / group, head r % group
      const int row_token = t * T + row_i;
      const bool have_row = row < T * a.group && q->tok0 + row_token < q->n;
      const int lim = (have_row ? piece_limit(a, *q, q->tok0 + row_token) : 0) - q->t0 * kKeyTile - hf * 64;  // keys of this half, counted from tile t0
      const int lim_first = piece_limit(a, *q, q->tok0 + t * T) - q->t0 * kKeyTile - hf * 64;  // the stream's first row sees fewest keys
      float row_unit = a.scale_log2;  // from S to logits in log2
      float m_ref = kNoMax;
      if (mode == kUseMaxima && n_mine > 0)  // what the pass before this one left
        m_ref = fmaxf(bars->left[(turn & 1) ^ 1][t][0][row], bars->left[(turn & 1) ^ 1][t][1][row]) - kLift;
      if constexpr (kFp8) {
        if (n_mine > 0) {
          ok = wait(bars->q_full[t], own & 1, kTileWaitQFull);
          if (!ok) break;
          // The thread's half row of Q into fp16, in place: the row's largest becomes 2^4 .. 2^5, so the halves' threads tell
          // each other the largest they have.
          const uint32_t src = q_smem + t * kTileBytes + hf * kTileHalf + row * 128, swz = row & 7;
          uint4 w[8];
          uint32_t m = 0;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            ld_shared_v4(src + ((x ^ swz) << 4), w[x]);
            m = __vmaxu2(m, __vmaxu2(__vmaxu2(w[x].x & 0x7FFF7FFFu, w[x].y & 0x7FFF7FFFu), __vmaxu2(w[x].z & 0x7FFF7FFFu, w[x].w & 0x7FFF7FFFu)));
          }
          m = max(m >> 16, m & 0xFFFFu);
          m = max(m, __float_as_uint(exchange(__uint_as_float(m))));
          if (!ok) break;
          const int e = max(static_cast<int>(m >> 7) - 127 - 4, -120);
          const float f = pow2_float(-e);
          row_unit *= pow2_float(e);
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const uint32_t in[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
            uint32_t o[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) o[z] = pack_f16x2(__uint_as_float(in[z] << 16) * f, __uint_as_float(in[z] & 0xFFFF0000u) * f);
            st_shared_v4(src + ((x ^ swz) << 4), o[0], o[1], o[2], o[3]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bars->q_ready[t]));
        }
      }
      float l_sum = 0.f;
      bool over = false;
#pragma unroll 1  // unrolled, it costs instruction cache: the whole kernel a sixth of its time on short pieces
      for (int it = 0; it < n_mine; ++it) {
        ok = wait(bars->s_full[t][hf], j & 1, kTileWaitS);
        if (!ok) break;
        tc_fence_after_sync();
        float c = row_unit;
        uint32_t e_at = 0;
        bool wide = false;
        if constexpr (kFp8) {
          const uint32_t slot = (n_before + it) % kInfoRing;
          const int kref = info[slot].kref;
          wide = info[slot].wide != 0;
          c = fminf(fmaxf(row_unit * __uint_as_float(static_cast<uint32_t>(kref) << 23), kLeastUnit), 3.0e38f);
          if (kref == 0) {  // every key has a factor of its own
            c = row_unit;
            e_at = smem_u32(&exps[slot][0][hf * 64]);
          }
        }
        // Where pieces are done again S is scaled first, so that the maxima and the terms are rounded alike: s c - m in one
        // step, with m rounded, is as far off as that rounding, and far more than the exponential takes for logits of 2^31.
        if (__builtin_expect(e_at != 0u || mode != kFirstTile, 0)) {
          scale_columns(s_addr, e_at, c);
          c = 1.f;
        }
        const bool partly = (it + 1) * kKeyTile - 64 > lim_first;
        const int valid = lim - it * kKeyTile;
        // 32 of the half's 64 keys at a time
        auto load = [&](uint32_t (&r)[32], int x) {
          tmem_ld32(s_addr + 32 * x, r);
          tmem_wait_ld();
          reg_fence32(r);
          if (partly) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= valid - 32 * x) r[i] = 0xFF800000u;  // -inf
          }
        };
        if (mode == kFindMaxima || (it == 0 && mode == kFirstTile)) {
#pragma unroll 1
          for (int x = 0; x < 2; ++x) {
            uint32_t r[32];
            load(r, x);
            float mx0 = fmax3(__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[2]));
            float mx1 = fmax3(__uint_as_float(r[3]), __uint_as_float(r[4]), __uint_as_float(r[5]));
#pragma unroll
            for (int i = 6; i < 30; i += 4) {
              mx0 = fmax3(mx0, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
              mx1 = fmax3(mx1, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
            }
            mx0 = fmax3(mx0, __uint_as_float(r[30]), __uint_as_float(r[31]));
            m_ref = fmaxf(m_ref, fmaxf(mx0, mx1) * c);  // a maximum of nothing but NaN: the reference stays finite
          }
          if (mode == kFirstTile) {
            m_ref = fmaxf(m_ref, exchange(m_ref)) - kLift;
            if (!ok) break;
            over = fabsf(m_ref) > 1.0e6f && m_ref > kNoMax;  // logits too large for s c - m in one step
          }
        }
        // P = 2^(s c - m), rounded once; the row sum keeps the unrounded terms
        float l_half = 0.f;
        const uint64_t c2 = pack2(c, c), nm2 = pack2(-m_ref, -m_ref);
        auto half = [&](auto pack) {
#pragma unroll 1
          for (int x = 0; x < 2; ++x) {
            uint32_t r[32], o[16];
            load(r, x);
            uint64_t acc0 = 0, acc1 = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float x0, x1;
              unpack2(fma2(pack2u(r[2 * i], r[2 * i + 1]), c2, nm2), x0, x1);
              const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
              if (i & 1) acc1 = add2(acc1, pack2(p0, p1));
              else acc0 = add2(acc0, pack2(p0, p1));
              o[i] = pack(p0, p1);
            }
            float a0, a1, a2, a3;
            unpack2(acc0, a0, a1);
            unpack2(acc1, a2, a3);
            l_half += (a0 + a1) + (a2 + a3);
            tmem_st16(s_addr + 16 * x, o);
          }
        };
        if (mode == kFindMaxima) {
          uint32_t o[16] = {};  // P = 0
          tmem_st16(s_addr, o);
          tmem_st16(s_addr + 16, o);
        } else if (kFp8 && !wide) {
          half([](float x, float y) { return pack_f16x2(x, y); });
        } else {
          half([](float x, float y) { return pack_bf16x2(x, y); });
        }
        l_sum += l_half;
        over |= !(l_half < kMostTerms);  // also infinities and NaN
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bars->p_full[t][hf]));
        ++j;
      }
      if (!ok) break;
      if constexpr (kFp8) n_before += q->n_tiles;
      if (n_mine > 0) ++own;
      if (mode == kFindMaxima) {  // the maxima stay where they were left
        exchange(m_ref);
        if (!ok) break;
      }
      if (mode == kFirstTile && over && have_row) atomicOr(&bars->redo, 1u << q->bit);
      // The helpers take it from here: O leaves tensor memory, row by row, while the next piece begins.  (Done here it took
      // 4.7 us per piece, the stores alone 2.5 at an SM's 26 GB/s to L2: as long as two and a half key tiles.)
      ok = n_fin == 0 || wait(bars->fin_free[t], (n_fin - 1) & 1, kTileWaitFinFree);
      if (!ok) break;
      ++n_fin;
      bars->sums[t][hf][row] = l_sum;
      if (hf == 0) bars->refs[t][row] = m_ref;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars->fin[t]));
    }
  }

  // ---- tear-down
  tc_fence_before_sync();
  __syncthreads();
  if (bars->abort_flag) {  // a wait gave up: give copies and MMAs in flight a bounded time to land
    if (threadIdx.x == 0 && a.c.status) atomicCAS(a.c.status, 0, static_cast<int>(bars->abort_flag | (blockIdx.x << 8)));
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == kIssuerWarp) {
    tc_fence_after_sync();
    tmem_dealloc(bars->tmem_base, 512);
  }
}

}  // namespace h3a
