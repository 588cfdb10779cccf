// Eviction from an 8-bit cache (block_cache.cuh) by accumulated attention weight: of the n finished blocks of a sequence, every
// layer and kv head keeps `keep`: its last `recent` ones and, among the others, those with the largest weight (of equal ones
// the lower index), in their order.  The kept blocks are copied, levels, scales and weight, to pages that the sequence does not
// use yet, so every block moves independently of every other and the old pages are as they were.
#include "block_cache.cuh"

using namespace iert;

namespace {

constexpr int SELECT_THREADS = 256;
constexpr int MOST_STAGED = 50 * 1024;       // blocks whose keys fit in shared memory

struct EvictParams {
  const float* weight;      // [layers][n_pages][kv_heads][per_page]
  const int* table;         // page table rows, `width` entries each
  const int* slots;         // row of sequence i (null: i)
  const int* lengths;       // [n] positions each sequence holds
  const int* new_pages;     // [n][new_width]
  int* kept;                // [layers][n][kv_heads][keep]: block numbers, -1 where the sequence has fewer
  int* shift;               // by row, or null: grows by the positions a sequence has lost
  int n, layers, n_pages, kv_heads, per_page, width, rows, new_width, keep, recent, max_blocks;
  int* err;
};

// A weight as a number whose order is the weights' order: NaN above everything, the two zeros alike.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int evict_row(const EvictParams& p, int i) {
  const int row = p.slots ? p.slots[i] : i;
  return row >= 0 && row < p.rows ? row : -1;
}
__device__ __forceinline__ int evict_page(const EvictParams& p, int row, int blk) {
  const int page = p.table[(size_t)row * p.width + blk / p.per_page];
  if (page < 0 || page >= p.n_pages) {
    atomicOr(p.err, IERT_ERR_PAGE_RANGE);
    return -1;
  }
  return page;
}
// Finished blocks of sequence i; -1 where it is longer than its row of the table.
__device__ __forceinline__ int evict_blocks(const EvictParams& p, int i) {
  const int length = max(p.lengths[i], 0);
  return length > (long long)p.width * p.per_page * BLK || length / BLK > p.max_blocks ? -1 : length / BLK;
}

// Which blocks stay: one CTA per (kv head, sequence, layer).  The keys stand in shared memory (STAGED; where they do not fit, in memory
// only, and are looked up again in each pass); the key of rank `need` is found eight bits at a time from counts of its leading digits (four
// passes, whole-number counts: the order of the additions cannot matter), then one ordered pass writes the numbers of the blocks above
// it, of as many equal ones as are missing, and of the last.
template <bool STAGED>
__global__ void __launch_bounds__(SELECT_THREADS) evict_select_kernel(EvictParams p) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[256], warp_gt[SELECT_THREADS / 32], warp_eq[SELECT_THREADS / 32], found[2];
  const int h = blockIdx.x, i = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int row = evict_row(p, i);
  int* kept = p.kept + (((size_t)layer * p.n + i) * p.kv_heads + h) * p.keep;
  const int nb = row < 0 ? -1 : evict_blocks(p, i);
  if (nb < 0 && tid == 0) atomicOr(p.err, IERT_ERR_PAGE_RANGE);      // (and the sequence is left as it is)
  if (nb <= p.keep) {                                    // nothing to choose
    for (int x = tid; x < p.keep; x += SELECT_THREADS) kept[x] = x < nb ? x : -1;
    return;
  }
  if (p.shift && h == 0 && layer == 0 && tid == 0) p.shift[row] += (nb - p.keep) * BLK;
  const int cand = nb - p.recent;                        // recent <= keep < nb
  int need = p.keep - p.recent;                          // this many of the first `cand`
  const float* w = p.weight + (size_t)layer * p.n_pages * p.kv_heads * p.per_page;
  auto look_up = [&](int x) {
    const int page = evict_page(p, row, x);
    return page < 0 ? 0u : weight_key(w[((size_t)page * p.kv_heads + h) * p.per_page + x % p.per_page]);
  };
  if (STAGED)
    for (int x = tid; x < cand; x += SELECT_THREADS) keys[x] = look_up(x);       // (read again by the thread that wrote it)
  auto key = [&](int x) { return STAGED ? keys[x] : look_up(x); };
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    for (int x = tid; x < 256; x += SELECT_THREADS) hist[x] = 0;
    __syncthreads();
    for (int x = tid; x < cand; x += SELECT_THREADS) {
      const uint32_t k = key(x);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (warp == 0) {                                     // the digit at which the count from above reaches `need`
      int mine = 0;
#pragma unroll
      for (int d = 0; d < 8; ++d) mine += hist[255 - (lane * 8 + d)];
      int before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      before -= mine;
      if (before < need && before + mine >= need) {
        int d = 0;
        while (before + hist[255 - (lane * 8 + d)] < need) before += hist[255 - (lane * 8 + d++)];
        found[0] = 255 - (lane * 8 + d);
        found[1] = need - before;
      }
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    need = found[1];                                     // among the keys that begin with `prefix`
    __syncthreads();
  }
  const bool any = p.keep > p.recent;
  int written = 0, equal = 0;                            // so far, over the whole block
  for (int base = 0; base < nb; base += SELECT_THREADS) {
    const int x = base + tid;
    const uint32_t k = x < cand && any ? key(x) : 0;
    const bool gt = (x < cand && any && k > prefix) || (x >= cand && x < nb), eq = x < cand && any && k == prefix;
    const unsigned bq = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) warp_eq[warp] = __popc(bq);
    __syncthreads();
    int rank = equal + __popc(bq & ((1u << lane) - 1));
    for (int v = 0; v < SELECT_THREADS / 32; ++v) {
      if (v < warp) rank += warp_eq[v];
      equal += warp_eq[v];
    }
    const bool take = gt || (eq && rank < need);
    const unsigned bt = __ballot_sync(0xffffffffu, take);
    if (lane == 0) warp_gt[warp] = __popc(bt);
    __syncthreads();
    int at = written + __popc(bt & ((1u << lane) - 1));
    for (int v = 0; v < SELECT_THREADS / 32; ++v) {
      if (v < warp) at += warp_gt[v];
      written += warp_gt[v];
    }
    if (take && at < p.keep) kept[at] = x;
    __syncthreads();
  }
}

struct CopyParams {
  uint8_t *k, *v;           // [layers][n_pages][kv_heads][page_tokens][head_dim]
  float *k_scale, *v_scale, *weight;
  int bytes;                // of a block's keys
};

// The copies: a warp per kept block (and one more per sequence, layer and head for the weight of the unfinished block, which the
// sequence keeps).  VEC: 16 bytes at a time.  Their bound is memory: 8 layers of 8 sequences of 4,096 positions, half of which stay
// (539 MB read and written), take 92 us with the choice in front, 5.9 TB/s; 32 layers of one sequence of 1,088 (135 MB) 28 us, of which the
// two starts, the choice and the chain kept -> page -> levels are about 8.  Copying after the choice in the same kernel would leave a CTA per
// head to copy all its blocks.
template <bool VEC>
__global__ void __launch_bounds__(256) evict_copy_kernel(EvictParams p, CopyParams q) {
  const int lane = threadIdx.x & 31, groups = p.keep / 8 + 1;       // eight kept blocks, neighbours where they go, to a block of threads
  const int lsh = blockIdx.x / groups, x = (blockIdx.x - lsh * groups) * 8 + (threadIdx.x >> 5);
  const int li = lsh / p.kv_heads, h = lsh - li * p.kv_heads, layer = li / p.n, i = li - layer * p.n;
  pdl_wait();                                            // the choice has been made
  if (x > p.keep) return;
  const int row = evict_row(p, i);
  if (row < 0) return;
  const int nb = evict_blocks(p, i);
  if (nb < 0) return;
  int from, to;
  const bool open = x == p.keep;
  if (open) {
    if (max(p.lengths[i], 0) % BLK == 0) return;
    from = nb;
    to = min(nb, p.keep);
  } else {
    from = p.kept[(size_t)lsh * p.keep + x];
    to = x;
    if (from < 0 || from >= nb) return;
  }
  if (to / p.per_page >= p.new_width) {                // no room for the unfinished block
    if (lane == 0) atomicOr(p.err, IERT_ERR_PAGE_RANGE);
    return;
  }
  const int src = evict_page(p, row, from), dst = p.new_pages[(size_t)i * p.new_width + to / p.per_page];
  if (src < 0) return;
  if (dst < 0 || dst >= p.n_pages) {
    if (lane == 0) atomicOr(p.err, IERT_ERR_PAGE_RANGE);
    return;
  }
  const size_t l0 = (size_t)layer * p.n_pages;
  const size_t a = ((l0 + src) * p.kv_heads + h) * p.per_page + from % p.per_page, z = ((l0 + dst) * p.kv_heads + h) * p.per_page + to % p.per_page;
  // lane 0 and, of a finished block, 1 and 2: weight and scales, on their way together with the levels
  float* small = lane == 0 ? q.weight : open || lane > 2 ? nullptr : lane == 1 ? q.k_scale : q.v_scale;
  const float was = small ? small[a] : 0.f;
  if (!open) {
    const uint8_t *ka = q.k + a * q.bytes, *va = q.v + a * q.bytes;
    uint8_t *kz = q.k + z * q.bytes, *vz = q.v + z * q.bytes;
    if (VEC) {
      const int n = q.bytes / 16;
      for (int j0 = lane; j0 < n; j0 += 128) {           // eight loads on their way before the first store
        uint4 r[8];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j0 + 32 * j < n) { r[2 * j] = __ldcs((const uint4*)ka + j0 + 32 * j); r[2 * j + 1] = __ldcs((const uint4*)va + j0 + 32 * j); }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j0 + 32 * j < n) { __stcs((uint4*)kz + j0 + 32 * j, r[2 * j]); __stcs((uint4*)vz + j0 + 32 * j, r[2 * j + 1]); }
      }
    } else {
      for (int j = lane; j < q.bytes; j += 32) { kz[j] = ka[j]; vz[j] = va[j]; }
    }
  }
  if (small) small[z] = was;
}

}  // namespace

// Two launches.  `max_blocks`: an upper bound on the sequences' finished blocks (sizes the shared memory).
IERT_API int iert_block_evict(void* k, void* v, float* k_scale, float* v_scale, float* weight, int layers, int n_pages, int kv_heads, int page_tokens,
                              int head_dim, const int* table, int width, int rows, const int* slots, const int* lengths, int n,
                              const int* new_pages, int new_width, int keep, int recent, int max_blocks, int* kept, int* shift, int* err,
                              cudaStream_t stream) {
  if (n <= 0 || layers <= 0) return IERT_OK;
  if (n_pages <= 0 || kv_heads <= 0 || page_tokens <= 0 || page_tokens % BLK || head_dim <= 0 || width <= 0 || rows <= 0 || keep <= 0 || recent < 0 ||
      recent > keep || max_blocks <= 0 || n > 65535 || layers > 65535 || (long long)new_width * page_tokens < (long long)keep * BLK)
    return IERT_BAD_ARGUMENT;
  const long long grid = (long long)layers * n * kv_heads * (keep / 8 + 1);          // of the copies; in front of both launches: the first one changes `shift`
  if (grid > 0x7fffffffLL) return IERT_BAD_ARGUMENT;
  const bool staged = max_blocks <= MOST_STAGED;
  const size_t smem = staged ? (size_t)max_blocks * sizeof(uint32_t) : 0;
  EvictParams p = {};
  p.weight = weight; p.table = table; p.slots = slots; p.lengths = lengths; p.new_pages = new_pages; p.kept = kept; p.shift = shift;
  p.n = n; p.layers = layers; p.n_pages = n_pages; p.kv_heads = kv_heads; p.per_page = page_tokens / BLK; p.width = width; p.rows = rows;
  p.new_width = new_width; p.keep = keep; p.recent = recent; p.max_blocks = max_blocks; p.err = err;
  if (smem > 40 * 1024 && !shared_memory_up_to<evict_select_kernel<true>>(MOST_STAGED * sizeof(uint32_t))) return iert_check_launch("block_evict (shared memory)");
  launch_dep(staged ? evict_select_kernel<true> : evict_select_kernel<false>, dim3(kv_heads, n, layers), dim3(SELECT_THREADS), smem, stream, p);
  const int status = iert_check_launch("block_evict (choice)");
  if (status) return status;
  CopyParams q = {(uint8_t*)k, (uint8_t*)v, k_scale, v_scale, weight, BLK * head_dim};
  const bool vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0;        // (a block is 16 x head_dim bytes)
  launch_dep(vec ? evict_copy_kernel<true> : evict_copy_kernel<false>, dim3((unsigned)grid), dim3(256), 0, stream, p, q);
  return iert_check_launch("block_evict (copy)");
}
