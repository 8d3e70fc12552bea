// C-ABI entry points of the paged K/V cache: argument validation and kernel launches.  Contracts live in include/h3attn.h.
#include "../../include/h3attn.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>

#include "cache_attn_few.cuh"
#include "cache_attn_tile.cuh"

namespace {

constexpr int kMaxDevices = 64;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// rows can be moved 16 bytes at a time; what is only read may repeat a row (stride 0)
bool rows16(int64_t stride, int64_t elem, bool read_only = false) { return (stride > 0 || (read_only && stride == 0)) && (stride * elem) % 16 == 0; }

struct Device {
  int id = -1, sms = 0, major = 0;
};
int32_t current_device(Device* d) {
  static Device known[kMaxDevices];
  static std::mutex lock;
  int id = 0;
  if (cudaGetDevice(&id) != cudaSuccess || id < 0 || id >= kMaxDevices) return H3A_ERR_LAUNCH;
  std::lock_guard<std::mutex> g(lock);
  if (known[id].id < 0) {
    Device n;
    if (cudaDeviceGetAttribute(&n.major, cudaDevAttrComputeCapabilityMajor, id) != cudaSuccess ||
        cudaDeviceGetAttribute(&n.sms, cudaDevAttrMultiProcessorCount, id) != cudaSuccess)
      return H3A_ERR_LAUNCH;
    n.id = id;
    known[id] = n;
  }
  *d = known[id];
  return d->major == 10 ? H3A_OK : H3A_ERR_ARCH;
}

// Checks a cache (which the call writes to, or reads only) and a batch and fills the kernels' view of them.
int32_t cache_args(bool write, const h3a_cache* c, const h3a_cache_batch* b, int32_t* status, h3a::CacheArgs* a) {
  if (!c || !b || !c->k || !c->v || !b->pages || !b->lengths || !b->starts) return H3A_ERR_ARG;
  if (c->quantised != 0 && c->quantised != 1) return H3A_ERR_ARG;
  if (c->quantised ? (!c->k_exp || !c->v_exp) : (c->k_exp || c->v_exp)) return H3A_ERR_ARG;
  if (c->d != 128 || c->n_pages <= 0 || c->heads <= 0 || c->page_size <= 0 || c->page_size % 16 || c->page_size > 65536) return H3A_ERR_SHAPE;
  if (b->n_seqs <= 0 || b->max_pages <= 0 || b->rows <= 0) return H3A_ERR_SHAPE;
  if (static_cast<int64_t>(b->max_pages) * c->page_size > (1ll << 28)) return H3A_ERR_SHAPE;
  if (static_cast<int64_t>(b->rows) * 2 * c->heads >= (1ll << 31)) return H3A_ERR_SHAPE;
  if (b->pages_stride < 0) return H3A_ERR_ARG;
  const int64_t es = c->quantised ? 1 : 2;
  if (!aligned16(c->k) || !aligned16(c->v)) return H3A_ERR_ALIGN;
  const int64_t strides[2][3] = {{c->k_stride_page, c->k_stride_token, c->k_stride_head}, {c->v_stride_page, c->v_stride_token, c->v_stride_head}};
  for (auto& s : strides)
    for (int64_t x : s)
      if (!rows16(x, es)) return H3A_ERR_ALIGN;
  // an exponent byte that rows share can be read, but not take all their exponents
  for (int64_t x : {c->k_exp_stride_page, c->k_exp_stride_token, c->k_exp_stride_head, c->v_exp_stride_page, c->v_exp_stride_token, c->v_exp_stride_head})
    if (c->quantised && x < (write ? 1 : 0)) return H3A_ERR_ALIGN;
  std::memset(a, 0, sizeof(*a));
  a->pool[0] = static_cast<uint8_t*>(c->k);
  a->pool[1] = static_cast<uint8_t*>(c->v);
  for (int x = 0; x < 2; ++x) {
    a->page_bytes[x] = strides[x][0] * es;
    a->token_bytes[x] = strides[x][1] * es;
    a->head_bytes[x] = strides[x][2] * es;
  }
  a->exps[0] = c->k_exp;
  a->exps[1] = c->v_exp;
  a->exp_page[0] = c->k_exp_stride_page;
  a->exp_token[0] = c->k_exp_stride_token;
  a->exp_head[0] = c->k_exp_stride_head;
  a->exp_page[1] = c->v_exp_stride_page;
  a->exp_token[1] = c->v_exp_stride_token;
  a->exp_head[1] = c->v_exp_stride_head;
  a->pages = b->pages;
  a->pages_stride = b->pages_stride;
  a->lengths = b->lengths;
  a->starts = b->starts;
  a->n_seqs = b->n_seqs;
  a->max_pages = b->max_pages;
  a->n_pages = c->n_pages;
  a->page_size = c->page_size;
  a->by_page = h3a::FastDiv::of(c->page_size);
  a->kv_heads = c->heads;
  a->rows = b->rows;
  a->status = status;
  return H3A_OK;
}

int32_t move_rows(bool write, const h3a_cache* c, const h3a_cache_batch* b, void* k, int64_t k_sl, int64_t k_sh, void* v, int64_t v_sl,
                  int64_t v_sh, int32_t* status, void* stream) {
  h3a::RowsArgs a;
  int32_t rc = cache_args(write, c, b, status, &a.c);
  if (rc != H3A_OK) return rc;
  if (!k || !v) return H3A_ERR_ARG;
  if (!aligned16(k) || !aligned16(v) || !rows16(k_sl, 2, write) || !rows16(k_sh, 2, write) || !rows16(v_sl, 2, write) || !rows16(v_sh, 2, write))
    return H3A_ERR_ALIGN;
  Device dev;
  if ((rc = current_device(&dev)) != H3A_OK) return rc;
  a.x[0] = static_cast<uint8_t*>(k);
  a.x[1] = static_cast<uint8_t*>(v);
  a.row_bytes[0] = k_sl * 2;
  a.head_bytes[0] = k_sh * 2;
  a.row_bytes[1] = v_sl * 2;
  a.head_bytes[1] = v_sh * 2;
  // Half-warps per token: one is the cheapest (a token is looked up once), but few tokens are spread over more of them,
  // up to a block's 16, and over further blocks, until about eight of them run on every SM.
  const int64_t want = 8ll * dev.sms;
  int per_token = 1;
  while (per_token < h3a::kRowGroups && b->rows * static_cast<int64_t>(per_token) < want && per_token < c->heads) per_token *= 2;
  const int64_t blocks_x = (b->rows + static_cast<int64_t>(h3a::kRowGroups / per_token) - 1) / (h3a::kRowGroups / per_token);
  const int64_t more = std::max<int64_t>(1, std::min(want / std::max<int64_t>(1, b->rows * static_cast<int64_t>(per_token)), static_cast<int64_t>(c->heads) / per_token));
  const dim3 grid(static_cast<unsigned>(blocks_x), static_cast<unsigned>(more));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (write) {
    if (c->quantised) h3a::cache_rows_kernel<true, true><<<grid, h3a::kRowThreads, 0, st>>>(a, per_token);
    else h3a::cache_rows_kernel<true, false><<<grid, h3a::kRowThreads, 0, st>>>(a, per_token);
  } else {
    if (c->quantised) h3a::cache_rows_kernel<false, true><<<grid, h3a::kRowThreads, 0, st>>>(a, per_token);
    else h3a::cache_rows_kernel<false, false><<<grid, h3a::kRowThreads, 0, st>>>(a, per_token);
  }
  return cudaGetLastError() == cudaSuccess ? H3A_OK : H3A_ERR_LAUNCH;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// x[..., row of 128]: outer dimensions with strides in bytes; a box of 128 bytes of a row, 128-byte swizzle
int32_t row_map(CUtensorMap* m, const void* ptr, bool codes, int n_outer, const int64_t* sizes, const int64_t* strides, const int* box_outer) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return H3A_ERR_DRIVER;
  cuuint64_t dims[4] = {128}, str[3];
  cuuint32_t box[4] = {codes ? 128u : 64u}, step[4] = {1, 1, 1, 1};
  for (int i = 0; i < n_outer; ++i) {
    dims[i + 1] = static_cast<cuuint64_t>(sizes[i]);
    str[i] = static_cast<cuuint64_t>(strides[i]);
    box[i + 1] = static_cast<cuuint32_t>(box_outer[i]);
  }
  return enc(m, codes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, n_outer + 1, const_cast<void*>(ptr), dims, str, box,
             step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? H3A_OK : H3A_ERR_LAUNCH;
}

// log2 of the units (a tile, or an item's set-up) below which a share is not worth a CTA
constexpr int kTileShareShift = 2, kFewShareShift = 1;
// Units for an item's set-up: Q on its way, the first tile's maxima, the last P V.  With one unit for it the tile kernel's CTAs
// with many items of a single key tile were the last to finish (prompts of 77 and 512 tokens: 138 us; 2: 122, 3: 125, 5: 127;
// bf16 115, 114, 104, 111).
constexpr int kTileSetUp = 3, kFewSetUp = 1;

// What a call of this shape launches.
struct AttnPlan {
  int item_rows = 0, item_tokens = 0, key_shift = 0, shares = 0;
  size_t bytes = 0;
};
AttnPlan attn_plan(const h3a_cache_attn_params* p, int sms) {
  AttnPlan n;
  const int group = p->heads / p->cache.heads;
  // query rows per K/V head: of the longest sequence, if the caller says so, else of the average one (the numbers
  // themselves are known on the device only); either kernel computes any batch
  const int64_t tokens = p->max_new > 0 ? p->max_new : (static_cast<int64_t>(p->batch.rows) + p->batch.n_seqs - 1) / p->batch.n_seqs;
  const int64_t rows = tokens * group;
  if (rows > h3a::kFewRows && group <= 128) {
    n.item_rows = h3a::kTileRows;
    n.item_tokens = 2 * (128 / group);
    n.key_shift = h3a::kTileKeyShift;
    n.shares = sms;
  } else {
    n.item_rows = rows <= 8 ? 8 : h3a::kFewRows;
    n.key_shift = h3a::kFewKeyShift;
    n.shares = sms * (rows <= 8 ? (p->cache.quantised ? h3a::kFewBlocksPerSm<true, 1> : h3a::kFewBlocksPerSm<false, 1>)
                                : (p->cache.quantised ? h3a::kFewBlocksPerSm<true, 2> : h3a::kFewBlocksPerSm<false, 2>));
  }
  n.bytes = static_cast<size_t>(n.shares) * (h3a::kDescInts * sizeof(int) + 2ull * n.item_rows * (h3a::kCacheDim + 2) * sizeof(float));
  return n;
}

template <bool kFp8, int kNT>
int32_t launch_few(const h3a::CacheAttnArgs& a, int shares, const Device& dev, cudaStream_t st) {
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  constexpr int kSmem = sizeof(h3a::FewSmem<kNT>);
  std::call_once(once[dev.id], [&] {
    err[dev.id] = cudaFuncSetAttribute(h3a::cache_attn_few_kernel<kFp8, kNT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (err[dev.id] != cudaSuccess) return H3A_ERR_LAUNCH;
  h3a::cache_attn_few_kernel<kFp8, kNT><<<shares, h3a::kFewThreads, kSmem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? H3A_OK : H3A_ERR_LAUNCH;
}

template <bool kFp8>
int32_t launch_tile(const h3a_cache_attn_params* p, const h3a::CacheAttnArgs& a, int shares, const Device& dev, cudaStream_t st) {
  static std::once_flag once[kMaxDevices];
  static cudaError_t err[kMaxDevices];
  std::call_once(once[dev.id], [&] {
    err[dev.id] = cudaFuncSetAttribute(h3a::cache_attn_tile_kernel<kFp8>, cudaFuncAttributeMaxDynamicSharedMemorySize, h3a::kTileSmemBytes);
  });
  if (err[dev.id] != cudaSuccess) return H3A_ERR_LAUNCH;
  CUtensorMap mq, mk, mv;
  const h3a_cache& c = p->cache;
  const int box_rows = std::min(128, c.page_size & -c.page_size);
  const int64_t q_sizes[2] = {p->heads, p->batch.rows}, q_strides[2] = {a.q_head_bytes, a.q_row_bytes};
  const int q_box[2] = {a.group, a.item_tokens / 2};
  int32_t rc = row_map(&mq, p->q, false, 2, q_sizes, q_strides, q_box);
  const int64_t sizes[3] = {c.page_size, c.heads, c.n_pages};
  const int box[3] = {box_rows, 1, 1};
  for (int x = 0; x < 2 && rc == H3A_OK; ++x) {
    const int64_t strides[3] = {a.c.token_bytes[x], a.c.head_bytes[x], a.c.page_bytes[x]};
    rc = row_map(x ? &mv : &mk, x ? c.v : c.k, kFp8, 3, sizes, strides, box);
  }
  if (rc != H3A_OK) return rc;
  h3a::cache_attn_tile_kernel<kFp8><<<shares, h3a::kTileThreads, h3a::kTileSmemBytes, st>>>(mq, mk, mv, box_rows, a);
  return cudaGetLastError() == cudaSuccess ? H3A_OK : H3A_ERR_LAUNCH;
}

int32_t launch_join(const h3a::CacheAttnArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;  // its launch overlaps the end of the kernel before it
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  // at most so many items: sequences, and as many more as their rows fill
  const int64_t rows = static_cast<int64_t>(a.c.rows) * a.group;
  const int64_t items = a.c.kv_heads * (a.c.n_seqs + std::max<int64_t>(0, rows - a.c.n_seqs) / a.item_rows);
  // ... in at most so many parts, of two units at least
  const int64_t parts = std::min<int64_t>(a.shares / items, static_cast<int64_t>(a.c.max_pages) * a.c.page_size >> (a.key_shift + a.share_shift));
  // More than the 16 parts that a warp takes at a time: one token over 131,072 keys, 8 heads on 1, 26 against 49 us; with
  // fewer the other is faster (over 1,023 keys, 8 heads: 10 against 12 us).
  if (a.item_tokens == 0 && parts > 16) {
    cfg.gridDim = dim3(static_cast<unsigned>(items), a.item_rows);
    cfg.blockDim = dim3(h3a::kWideWarps * 32);
    return cudaLaunchKernelEx(&cfg, h3a::cache_attn_join_wide_kernel, a) == cudaSuccess ? H3A_OK : H3A_ERR_LAUNCH;
  }
  // a warp per row where rows are few, and per two rows of larger items: 8 blocks per item instead of 32 left 20 items of
  // 252 rows in 18 parts to too few warps (chunks of 3 to 301 tokens: 53 against 39 us in all), 64 are not faster
  cfg.gridDim = dim3(a.shares, std::min(32, a.item_rows / h3a::kJoinRows));
  cfg.blockDim = dim3(h3a::kJoinRows * 32);
  const auto kernel = a.item_tokens > 0 ? h3a::cache_attn_join_kernel<4> : h3a::cache_attn_join_kernel<16>;
  return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? H3A_OK : H3A_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int32_t h3a_cache_write(const h3a_cache* cache, const h3a_cache_batch* batch, const void* k, int64_t k_stride_l, int64_t k_stride_h,
                        const void* v, int64_t v_stride_l, int64_t v_stride_h, int32_t* status_word, void* stream) {
  return move_rows(true, cache, batch, const_cast<void*>(k), k_stride_l, k_stride_h, const_cast<void*>(v), v_stride_l, v_stride_h,
                   status_word, stream);
}

int32_t h3a_cache_read(const h3a_cache* cache, const h3a_cache_batch* batch, void* k, int64_t k_stride_l, int64_t k_stride_h,
                       void* v, int64_t v_stride_l, int64_t v_stride_h, int32_t* status_word, void* stream) {
  return move_rows(false, cache, batch, k, k_stride_l, k_stride_h, v, v_stride_l, v_stride_h, status_word, stream);
}

int32_t h3a_cache_attn_workspace_bytes(const h3a_cache_attn_params* p, size_t* bytes) {
  if (!p || !bytes) return H3A_ERR_ARG;
  if (p->cache.heads <= 0 || p->heads <= 0 || p->heads % p->cache.heads || p->batch.rows <= 0 || p->batch.n_seqs <= 0) return H3A_ERR_SHAPE;
  Device dev;
  const int32_t rc = current_device(&dev);
  if (rc != H3A_OK) return rc;
  *bytes = attn_plan(p, dev.sms).bytes;
  return H3A_OK;
}

int32_t h3a_cache_attn(const h3a_cache_attn_params* p, void* stream) {
  if (!p || !p->q || !p->o || p->o == p->q) return H3A_ERR_ARG;  // a piece that is done twice reads its q again
  h3a::CacheAttnArgs a;
  std::memset(&a, 0, sizeof(a));
  int32_t rc = cache_args(false, &p->cache, &p->batch, p->status_word, &a.c);
  if (rc != H3A_OK) return rc;
  if (p->heads <= 0 || p->heads % p->cache.heads || static_cast<int64_t>(p->batch.rows) * p->heads >= (1ll << 31)) return H3A_ERR_SHAPE;
  if ((p->causal != 0 && p->causal != 1) || p->max_new < 0) return H3A_ERR_ARG;
  if (!aligned16(p->q) || !aligned16(p->o) || !rows16(p->q_stride_l, 2) || !rows16(p->q_stride_h, 2) || !rows16(p->o_stride_l, 2) ||
      !rows16(p->o_stride_h, 2))
    return H3A_ERR_ALIGN;
  Device dev;
  if ((rc = current_device(&dev)) != H3A_OK) return rc;
  const AttnPlan n = attn_plan(p, dev.sms);
  if (!p->workspace || p->workspace_bytes < n.bytes) return H3A_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(p->workspace) % 32) return H3A_ERR_ALIGN;
  a.q = static_cast<const uint8_t*>(p->q);
  a.q_row_bytes = p->q_stride_l * 2;
  a.q_head_bytes = p->q_stride_h * 2;
  a.o = static_cast<__nv_bfloat16*>(p->o);
  a.o_stride_l = p->o_stride_l;
  a.o_stride_h = p->o_stride_h;
  a.o_sectors = (reinterpret_cast<uintptr_t>(p->o) | static_cast<uintptr_t>(2 * p->o_stride_l) | static_cast<uintptr_t>(2 * p->o_stride_h)) % 32 == 0;
  a.lse = p->lse;
  a.heads = p->heads;
  a.group = p->heads / p->cache.heads;
  a.causal = p->causal;
  a.item_rows = n.item_rows;
  a.item_tokens = n.item_tokens;
  a.key_shift = n.key_shift;
  a.scale_log2 = (p->softmax_scale > 0.f ? p->softmax_scale : 1.0f / std::sqrt(128.0f)) * 1.4426950408889634f;
  a.desc = static_cast<int*>(p->workspace);
  a.part = reinterpret_cast<float*>(a.desc + h3a::kDescInts * n.shares);
  a.shares = n.shares;
  a.set_up = n.item_tokens > 0 ? kTileSetUp : kFewSetUp;
  a.share_shift = n.item_tokens > 0 ? kTileShareShift : kFewShareShift;
  a.by_group = h3a::FastDiv::of(a.group);
  a.by_item_rows = h3a::FastDiv::of(n.item_rows);
  a.by_item_tokens = h3a::FastDiv::of(std::max(1, n.item_tokens));
  a.wait_units = static_cast<uint32_t>(std::min<int64_t>((p->wait_limit_ns > 0 ? p->wait_limit_ns : 2000000000ll) >> 10, 0x7FFFFFFF));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n.item_tokens > 0)
    rc = p->cache.quantised ? launch_tile<true>(p, a, n.shares, dev, st) : launch_tile<false>(p, a, n.shares, dev, st);
  else if (n.item_rows == 8)
    rc = p->cache.quantised ? launch_few<true, 1>(a, n.shares, dev, st) : launch_few<false, 1>(a, n.shares, dev, st);
  else
    rc = p->cache.quantised ? launch_few<true, 2>(a, n.shares, dev, st) : launch_few<false, 2>(a, n.shares, dev, st);
  return rc == H3A_OK ? launch_join(a, st) : rc;
}

}  // extern "C"
