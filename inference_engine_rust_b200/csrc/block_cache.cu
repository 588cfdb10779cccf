// The cache in 8 bits (block_cache.cuh): writing a step's keys and values, one-token attention over it as the equations say (any
// head size up to 256; block_attention_tc.cu and block_attention_umma.cu have the tensor-core forms of the usual sizes).
#include <type_traits>

#include "block_cache.cuh"

using namespace iert;

namespace {

// ---------------------------------------------------------------------------------------
// Store: the keys and values of a step's tokens, positions [pos0, pos0 + q) of each sequence.  One CTA per (block of 16
// positions, kv head), half of it for the keys and half for the values.  The blocks of sequence s are the units [cu_q[s] / 16 + 2 s, ...): q
// tokens touch at most q / 16 + 2 blocks.  A step reads and writes each number once, and few tokens take the time of one chain of loads: so a
// thread asks for all its numbers (eight at a time, `RUNS` runs of them), keeps them in registers over the search for the
// largest, and writes their levels; the page is looked up while they are on their way.  2,048 tokens of 8 heads of 128 take 6 us (38 with two
// passes of single numbers), 16,001 of 4 heads of 64, 25 MB, 12, which is the time to issue 9.4 M warp instructions (2.5 of 4 a cycle): about 36 a
// number, most of them a CTA's own setup and the levels' two roundings; two heads of 64 a CTA, with half the setup, took 15.
constexpr int STORE_THREADS = 128, HALF = STORE_THREADS / 2;

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 f = __bfloat1622float2(h[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}
__device__ __forceinline__ void save8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void save8(__nv_bfloat16* p, const float (&x)[8]) {
  uint4 raw;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);       // (exact: they were bfloat16)
  *reinterpret_cast<uint4*>(p) = raw;
}

// RUNS > 0: head sizes up to 32 RUNS, multiples of eight, all rows 16-byte aligned; HD > 0: that size alone, so that places in rows are
// found without divisions.  0, 0: any.
template <int FMT, typename T, int RUNS, int HD>
__global__ void __launch_bounds__(STORE_THREADS) block_store_kernel(const T* __restrict__ qkv, int heads, IertBatchView b, IertBlockView c, int* __restrict__ err) {
  __shared__ uint32_t red[STORE_THREADS / 32];
  pdl_launch_dependents();
  const int u = blockIdx.x, h = blockIdx.y, hd = HD ? HD : c.head_dim;
  int lo = 0, hi = b.n_seqs;                           // the last sequence whose units start at or below u
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.cu_q[mid] / BLK + 2 * mid <= u) lo = mid; else hi = mid;
  }
  const int s = lo, slot = block_slot(c, b, s, err);
  if (slot < 0 || b.pos0[s] < 0) { pdl_wait(); return; }     // (a kernel that ends before the one in front of it would let the next one pass both)
  const int p0 = b.pos0[s], q0 = b.cu_q[s], end = p0 + b.cu_q[s + 1] - q0;
  const int first = p0 / BLK, blk = first + u - (q0 / BLK + 2 * s), open = end / BLK;     // `open`: the block that stays unfinished, if any
  pdl_wait();
  if (blk * BLK >= end || end == p0) return;
  const long long ld = (long long)(heads + 2 * c.kv_heads) * hd;
  const size_t t_off = ((size_t)slot * c.kv_heads + h) * BLK * hd;
  const int v = threadIdx.x / HALF, me = threadIdx.x % HALF;                              // keys or values
  const T* rows = qkv + (long long)q0 * ld + (long long)(heads + v * c.kv_heads + h) * hd;
  T* tail = (T*)(v ? c.tail_v : c.tail_k) + t_off;
  const int per_page = c.page_tokens / BLK;
  auto one = [&](int x) {
    const int base = x * BLK, n_old = max(0, p0 - base);       // rows that are in the tail already
    const int pg = x / per_page, in_page = x - pg * per_page;
    const bool whole = x < open, stays = whole && x + c.ring_pages * per_page >= open;
    // a ring keeps its latest blocks only: those that a later block of this step takes the place of are not written
    if (whole && !stays) return;                               // (a ring keeps no weights)
    const T* fresh = rows + (long long)(max(p0, base) - p0) * ld;
    const int n = (whole ? BLK : end - base) * hd;
    auto source = [&](int i) { const int r = i / hd; return r < n_old ? tail + i : fresh + (long long)(r - n_old) * ld + (i - r * hd); };
    float val[RUNS > 0 ? RUNS : 1][8];
    if constexpr (RUNS > 0) {
#pragma unroll
      for (int k = 0; k < RUNS; ++k) {
        const int i = (me + k * HALF) * 8;
        if (i < n) load8(source(i), val[k]);
      }
    }
    // (looked up while the numbers are on their way)
    const int page = whole || c.weight ? block_page(c, slot, pg, err) : -1;
    const size_t at = page >= 0 ? ((size_t)page * c.kv_heads + h) * per_page + in_page : 0;
    if (page >= 0 && c.weight && base >= p0 && threadIdx.x == 0) c.weight[at] = 0.f;
    if (whole && page < 0) return;
    uint8_t* levels = (uint8_t*)(v ? c.v : c.k) + at * BLK * hd;
    if (!whole) {
      if constexpr (RUNS > 0) {
#pragma unroll
        for (int k = 0; k < RUNS; ++k) {
          const int i = (me + k * HALF) * 8;
          if (i < n && i / hd >= n_old) save8(tail + i, val[k]);
        }
      } else {
        for (int i = n_old * hd + me; i < n; i += HALF) tail[i] = *source(i);
      }
      return;
    }
    uint32_t largest = 0;
    if constexpr (RUNS > 0) {
#pragma unroll
      for (int k = 0; k < RUNS; ++k)
        if ((me + k * HALF) * 8 < n)
#pragma unroll
          for (int e = 0; e < 8; ++e) largest = max(largest, abs_bits(val[k][e]));
    } else {
      for (int i = me; i < n; i += HALF) largest = max(largest, abs_bits(to_f32(*source(i))));
    }
    largest = __reduce_max_sync(0xffffffffu, largest);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = largest;
    __syncthreads();
    const float scale = block_scale<FMT>(max(red[2 * v], red[2 * v + 1])), inv = inverse_of_scale(scale);
    if constexpr (RUNS > 0) {
#pragma unroll
      for (int k = 0; k < RUNS; ++k) {
        const int i = (me + k * HALF) * 8;
        if (i >= n) break;
        *reinterpret_cast<uint2*>(levels + i) = make_uint2(to_levels4<FMT>(&val[k][0], scale, inv), to_levels4<FMT>(&val[k][4], scale, inv));
      }
    } else {
      for (int i = me; i < n; i += HALF) levels[i] = to_level<FMT>(to_f32(*source(i)), scale);
    }
    if (me == 0) (v ? c.v_scale : c.k_scale)[at] = scale;
  };
  // the tail is read by the first block and written by the unfinished one: the same CTA does them one after the other
  const bool together = p0 % BLK != 0 && first < open;
  if (together && blk == open) return;
  one(blk);
  if (together && blk == first && open * BLK < end) {
    __syncthreads();
    one(open);
  }
}

// ---------------------------------------------------------------------------------------
// One-token attention, plain: a CTA per (sequence, kv head), eight query heads of the group at a time, fp32 throughout.  A warp
// takes every eighth block, its lanes the dimensions; a block's sixteen scores are reduced across the lanes one by one.
constexpr int GH = 8, MAXD = 8;                 // heads at a time; dimensions per lane (head sizes up to 256)

struct BlockAttentionParams {
  const void* qkv;
  void* out;
  float* part;                 // scratch [T][heads][blocks]: base-2 logarithm of a block's unnormalised weight
  float* weight_out;
  int heads, blocks;
  float scale_log2e;
  const float* inv_freq;       // rope != 0: the kernel rotates queries and the new key itself
  int rope, rotary_dim, pairing;
  float rot_mul;
  int* err;
};

// Element d of a head rotated by the angles in cs = [cos | sin] of rotary_dim / 2 pairs.
template <typename T>
__device__ __forceinline__ float rotated(const T* src, int d, int rotary_dim, int pairing, const float* cs) {
  const float x = to_f32(src[d]);
  if (d >= rotary_dim) return x;
  const int half = rotary_dim / 2;
  const bool second = pairing == IERT_PAIR_HALF ? d >= half : d & 1;
  const int k = pairing == IERT_PAIR_HALF ? (second ? d - half : d) : d >> 1;
  const float y = to_f32(src[pairing == IERT_PAIR_HALF ? (second ? d - half : d + half) : d ^ 1]);
  return second ? y * cs[half + k] + x * cs[k] : x * cs[k] - y * cs[half + k];
}

template <int FMT, typename T>
__global__ void __launch_bounds__(256) block_attention_plain_kernel(BlockAttentionParams p, IertBatchView b, IertBlockView c) {
  extern __shared__ float sm[];
  constexpr int WARPS = 8;
  __shared__ uint32_t red[WARPS];
  const int hd = c.head_dim;
  float* cs = sm;                               // [hd] cos, sin
  float* qs = cs + hd;                          // [GH][hd] queries
  float* os = qs + GH * hd;                     // [WARPS][GH][hd]
  float* ml = os + WARPS * GH * hd;             // [WARPS][GH][2]
  pdl_launch_dependents();
  const int kvh = blockIdx.x, t = blockIdx.y, group = p.heads / c.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = sequence_of_token(b, t);
  int slot = block_slot(c, b, s, p.err);
  if (slot >= 0 && !block_reaches(c, b.pos0[s], p.err)) slot = -1;
  pdl_wait();
  T* out = (T*)p.out + ((size_t)t * p.heads + (size_t)kvh * group) * hd;
  if (slot < 0) {
    for (int i = threadIdx.x; i < group * hd; i += blockDim.x) out[i] = from_f32<T>(0.f);
    return;
  }
  const int pos = b.pos0[s], blk = pos / BLK, base = blk * BLK, per_page = c.page_tokens / BLK;
  const T* row = (const T*)p.qkv + (size_t)t * (size_t)(p.heads + 2 * c.kv_heads) * hd;
  const size_t t_off = ((size_t)slot * c.kv_heads + kvh) * BLK * hd;
  T *tk = (T*)c.tail_k + t_off, *tv = (T*)c.tail_v + t_off;
  if (p.rope) {
    const float where = (float)(pos + (c.shift ? c.shift[slot] : 0));
    for (int k = threadIdx.x; k < p.rotary_dim / 2; k += blockDim.x) {
      float sn, co;
      sincosf(where * p.inv_freq[k], &sn, &co);
      cs[k] = co * p.rot_mul;
      cs[p.rotary_dim / 2 + k] = sn * p.rot_mul;
    }
    __syncthreads();
  }
  // the step's own key and value join the tail
  const T *kn = row + (size_t)(p.heads + kvh) * hd, *vn = row + (size_t)(p.heads + c.kv_heads + kvh) * hd;
  for (int d = threadIdx.x; d < hd; d += blockDim.x) {
    tk[(pos - base) * hd + d] = p.rope ? from_f32<T>(rotated(kn, d, p.rotary_dim, p.pairing, cs)) : kn[d];
    tv[(pos - base) * hd + d] = vn[d];
  }
  __syncthreads();
  const int j_min = iert_first_visible(pos, c.window, 0);
  const int b_lo = j_min / BLK;
  for (int g0 = 0; g0 < group; g0 += GH) {
    const int n_g = min(GH, group - g0), head0 = kvh * group + g0;
    __syncthreads();
    for (int i = threadIdx.x; i < n_g * hd; i += blockDim.x) {
      const T* q = row + (size_t)(head0 + i / hd) * hd;
      qs[i] = p.rope ? to_f32(from_f32<T>(rotated(q, i % hd, p.rotary_dim, p.pairing, cs))) : to_f32(q[i % hd]);
    }
    __syncthreads();
    float o[GH][MAXD], m[GH], l[GH];
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      m[g] = -INFINITY; l[g] = 0.f;
#pragma unroll
      for (int e = 0; e < MAXD; ++e) o[g][e] = 0.f;
    }
    for (int x = b_lo + warp; x <= blk; x += WARPS) {
      const bool tail = x == blk;
      const int page = tail ? 0 : block_page(c, slot, x * BLK / c.page_tokens, p.err);
      if (page < 0) continue;
      const size_t at = ((size_t)page * c.kv_heads + kvh) * per_page + x % per_page;
      const uint8_t *kq = (const uint8_t*)c.k + at * BLK * hd, *vq = (const uint8_t*)c.v + at * BLK * hd;
      const float ks = tail ? 1.f : c.k_scale[at], vs = tail ? 1.f : c.v_scale[at];
      const int r_lo = max(0, j_min - x * BLK), r_hi = min(BLK - 1, pos - x * BLK);
      float sum[GH];                            // the block's weights relative to the running maximum
#pragma unroll
      for (int g = 0; g < GH; ++g) sum[g] = 0.f;
      for (int r = r_lo; r <= r_hi; ++r) {
        float kd[MAXD], vd[MAXD];
#pragma unroll
        for (int e = 0; e < MAXD; ++e) {
          const int d = lane + 32 * e;
          kd[e] = d >= hd ? 0.f : tail ? to_f32(tk[r * hd + d]) : from_level<FMT>(kq[r * hd + d]) * ks;
          vd[e] = d >= hd ? 0.f : tail ? to_f32(tv[r * hd + d]) : from_level<FMT>(vq[r * hd + d]) * vs;
        }
#pragma unroll
        for (int g = 0; g < GH; ++g) {
          if (g >= n_g) break;
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < MAXD; ++e)
            if (lane + 32 * e < hd) dot = fmaf(qs[g * hd + lane + 32 * e], kd[e], dot);
          const float sc = warp_sum(dot) * p.scale_log2e;
          // a score of -infinity (or NaN) must not make 0 * infinity of what is there already
          const float mx = fmaxf(m[g], sc);
          const float alpha = m[g] == -INFINITY ? 0.f : exp2f(m[g] - mx);
          const float pr = mx == -INFINITY ? (sc == sc ? 0.f : sc) : exp2f(sc - mx);
          m[g] = mx;
          l[g] = l[g] * alpha + pr;
          sum[g] = sum[g] * alpha + pr;
#pragma unroll
          for (int e = 0; e < MAXD; ++e) o[g][e] = fmaf(pr, vd[e], o[g][e] * alpha);
        }
      }
      if (c.weight && lane == 0) {
#pragma unroll
        for (int g = 0; g < GH; ++g)
          if (g < n_g) p.part[((size_t)t * p.heads + head0 + g) * p.blocks + x] = m[g] + log2f(sum[g]);
      }
    }
    // merge the warps in warp order
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      if (g >= n_g) break;
#pragma unroll
      for (int e = 0; e < MAXD; ++e)
        if (lane + 32 * e < hd) os[(warp * GH + g) * hd + lane + 32 * e] = o[g][e];
      if (lane == 0) { ml[(warp * GH + g) * 2] = m[g]; ml[(warp * GH + g) * 2 + 1] = l[g]; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n_g * hd; i += blockDim.x) {
      const int g = i / hd, d = i % hd;
      float mm = -INFINITY, ll = 0.f, acc = 0.f;
      for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, ml[(w * GH + g) * 2]);
      for (int w = 0; w < WARPS; ++w) {
        const float mw = ml[(w * GH + g) * 2], f = mw == -INFINITY ? 0.f : exp2f(mw - mm);
        ll += f * ml[(w * GH + g) * 2 + 1];
        acc += f * os[(w * GH + g) * hd + d];
      }
      out[(size_t)g0 * hd + i] = from_f32<T>(ll == 0.f ? 0.f : acc / ll);
    }
    if (c.weight) {
      // weight of block x: sum over the group's heads (in their order) of 2^(part - lse)
      for (int x = b_lo + threadIdx.x; x <= blk; x += blockDim.x) {
        const int page = block_page(c, slot, x * BLK / c.page_tokens, p.err);
        if (page < 0) continue;
        const size_t at = ((size_t)page * c.kv_heads + kvh) * per_page + x % per_page;
        float w = g0 > 0 ? p.weight_out[at] : (x == blk && pos == base) ? 0.f : c.weight[at];
        for (int g = 0; g < n_g; ++g) {
          float mm = -INFINITY, ll = 0.f;
          for (int v = 0; v < WARPS; ++v) mm = fmaxf(mm, ml[(v * GH + g) * 2]);
          for (int v = 0; v < WARPS; ++v) ll += ml[(v * GH + g) * 2] == -INFINITY ? 0.f : exp2f(ml[(v * GH + g) * 2] - mm) * ml[(v * GH + g) * 2 + 1];
          w += exp2f(p.part[((size_t)t * p.heads + head0 + g) * p.blocks + x] - mm) / ll;
        }
        p.weight_out[at] = w;
      }
    }
  }
  if (pos - base == BLK - 1) {                  // the block is complete: from the next step on it is read in 8 bits
    __syncthreads();
    const int page = block_page(c, slot, base / c.page_tokens, p.err);
    if (page >= 0) {
      const size_t at = ((size_t)page * c.kv_heads + kvh) * per_page + blk % per_page;
      finish_block<FMT>(tk, hd, (uint8_t*)c.k + at * BLK * hd, c.k_scale + at, red);
      finish_block<FMT>(tv, hd, (uint8_t*)c.v + at * BLK * hd, c.v_scale + at, red);
    }
  }
}

bool view_ok(const IertBlockView& c) {
  return c.n_slots > 0 && c.table_width > 0 && c.ring_pages > 0 && c.ring_pages <= c.table_width && c.n_pages > 0 && c.kv_heads > 0 && c.head_dim > 0 &&
         c.page_tokens > 0 && c.page_tokens % BLK == 0 && c.window >= 0 && (c.format == IERT_LEVEL_INT8 || c.format == IERT_LEVEL_E4M3) &&
         (c.tail_dtype == IERT_F32 || c.tail_dtype == IERT_BF16);
}

}  // namespace

IERT_API int iert_block_store(const void* qkv, int heads, const IertBatchView* batch, const IertBlockView* view, int* err, cudaStream_t stream) {
  if (batch->n_tokens <= 0 || batch->n_seqs <= 0) return IERT_OK;
  if (!view_ok(*view) || heads <= 0) return IERT_BAD_ARGUMENT;
  if (view->kv_heads > 65535) return IERT_BAD_ARGUMENT;
  const dim3 grid(batch->n_tokens / BLK + 2 * batch->n_seqs + 1, view->kv_heads);
  const int hd = view->head_dim;
  const bool vec = hd % 8 == 0 && hd <= 256 &&
                   ((uintptr_t)qkv | (uintptr_t)view->k | (uintptr_t)view->v | (uintptr_t)view->tail_k | (uintptr_t)view->tail_v) % 16 == 0;
  auto go = [&](auto fmt, auto* rows) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(rows)>>;
    constexpr int FMT = decltype(fmt)::value;
    auto with = [&](auto kernel) { launch_dep(kernel, grid, dim3(STORE_THREADS), 0, stream, rows, heads, *batch, *view, err); };
    if (!vec) with(block_store_kernel<FMT, T, 0, 0>);
    else if (hd == 64) with(block_store_kernel<FMT, T, 2, 64>);
    else if (hd == 128) with(block_store_kernel<FMT, T, 4, 128>);
    else with(block_store_kernel<FMT, T, 8, 0>);
  };
  using I8 = std::integral_constant<int, IERT_LEVEL_INT8>;
  using E4 = std::integral_constant<int, IERT_LEVEL_E4M3>;
  if (view->tail_dtype == IERT_F32) {
    if (view->format == IERT_LEVEL_INT8) go(I8(), (const float*)qkv); else go(E4(), (const float*)qkv);
  } else {
    if (view->format == IERT_LEVEL_INT8) go(I8(), (const __nv_bfloat16*)qkv); else go(E4(), (const __nv_bfloat16*)qkv);
  }
  return iert_check_launch("block_store");
}

static int block_attention_plain(const void* qkv, void* out, const IertBatchView* batch, const IertBlockView* view, int heads, float scale, float* part,
                                 float* weight_out, const float* inv_freq, int rotary_dim, int pairing, float rot_mul, int* err, cudaStream_t stream) {
  if (!view_ok(*view) || heads <= 0 || heads % view->kv_heads || view->head_dim > 32 * MAXD || batch->n_tokens != batch->n_seqs ||
      batch->n_seqs > 65535 || (view->weight && (view->window || !part || !weight_out)) ||
      (inv_freq && (rotary_dim < 0 || rotary_dim > view->head_dim || (rotary_dim & 1) || (pairing != IERT_PAIR_HALF && pairing != IERT_PAIR_INTERLEAVED))))
    return IERT_BAD_ARGUMENT;
  BlockAttentionParams p = {};
  p.qkv = qkv; p.out = out; p.part = part; p.weight_out = weight_out;
  p.heads = heads; p.blocks = view->table_width * (view->page_tokens / BLK);
  p.scale_log2e = scale * 1.44269504088896340736f;
  p.inv_freq = inv_freq; p.rope = inv_freq != nullptr; p.rotary_dim = rotary_dim; p.pairing = pairing; p.rot_mul = rot_mul; p.err = err;
  const int hd = view->head_dim;
  auto bytes = [](size_t d) { return sizeof(float) * (d + GH * d + 8 * GH * d + 8 * GH * 2); };
  const size_t smem = bytes(hd);
  const dim3 grid(view->kv_heads, batch->n_seqs);
  auto go = [&](auto fmt, auto* tail) {
    constexpr auto kernel = block_attention_plain_kernel<decltype(fmt)::value, std::remove_pointer_t<decltype(tail)>>;
    if (smem > 40 * 1024 && !shared_memory_up_to<kernel>(bytes(32 * MAXD))) return iert_check_launch("block_attention_plain (shared memory)");
    launch_dep(kernel, grid, dim3(256), smem, stream, p, *batch, *view);
    return iert_check_launch("block_attention_plain");
  };
  using I8 = std::integral_constant<int, IERT_LEVEL_INT8>;
  using E4 = std::integral_constant<int, IERT_LEVEL_E4M3>;
  if (view->tail_dtype == IERT_F32) return view->format == IERT_LEVEL_INT8 ? go(I8(), (float*)nullptr) : go(E4(), (float*)nullptr);
  return view->format == IERT_LEVEL_INT8 ? go(I8(), (__nv_bfloat16*)nullptr) : go(E4(), (__nv_bfloat16*)nullptr);
}

// `plain`: the kernel above alone.  Else the first that takes the case: tcgen05 (`splits`, `groups`), mma.sync (`splits`), and with `splits` 0 the one above.
IERT_API int iert_block_attention(const void* qkv, void* out, const IertBatchView* batch, const IertBlockView* view, int heads, float scale, float* scratch,
                                  float* weight_out, const float* inv_freq, int rotary_dim, int pairing, float rot_mul, int plain, int splits, int groups,
                                  int* err, cudaStream_t stream) {
  if (batch->n_tokens <= 0) return IERT_OK;
  if (!plain) {
    int status = block_attention_umma(qkv, out, batch, view, heads, scale, scratch, weight_out, inv_freq, rotary_dim, pairing, rot_mul, splits, groups, err, stream);
    if (status == IERT_BAD_ARGUMENT)
      status = block_attention_tc(qkv, out, batch, view, heads, scale, scratch, weight_out, inv_freq, rotary_dim, pairing, rot_mul, splits, err, stream);
    if (status != IERT_BAD_ARGUMENT || splits) return status;
  }
  return block_attention_plain(qkv, out, batch, view, heads, scale, scratch, weight_out, inv_freq, rotary_dim, pairing, rot_mul, err, stream);
}
