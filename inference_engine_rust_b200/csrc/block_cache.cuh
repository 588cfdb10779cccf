// A layer's keys and values held in 8 bits.  A block is 16 consecutive positions of one kv head: its 16 x head_dim keys share
// one fp32 scale and its values another; a level q (int8, or e4m3) stands for q * scale.  A block is written once, when its
// sixteenth position has arrived, from the numbers as they came (scale = max |x| / 127 or / 448): no number is rounded twice and
// what a block holds does not depend on how its positions arrived.  Until then a sequence's newest positions, fewer than 16,
// stand in `tail` in the run's own type.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

enum : int { IERT_LEVEL_INT8 = 0, IERT_LEVEL_E4M3 = 1 };

//   k, v             : levels [n_pages][kv_heads][page_tokens][head_dim]
//   k_scale, v_scale : [n_pages][kv_heads][page_tokens / 16]
//   weight           : accumulated attention weight of each block, laid out as the scales, or null (not kept)
//   tail_k, tail_v   : [n_slots][kv_heads][16][head_dim] of `tail_dtype`
//   page_table       : [n_slots][table_width]; page b of a sequence is entry b % ring_pages of its row
//   shift            : [n_slots] or null: positions a sequence has lost to eviction, i.e. how far the position of its row j
//                      (what a rotation turns by) lies above j
//   window           : 0 = every earlier position is visible; W > 0 = the last W, the current one included
struct IertBlockView {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  float* weight;
  void* tail_k;
  void* tail_v;
  const int* page_table;
  const int* shift;
  int n_slots;
  int table_width;
  int ring_pages;
  int n_pages;
  int kv_heads;
  int head_dim;
  int page_tokens;
  int window;
  int format;
  int tail_dtype;
};

// One-token attention on tcgen05 (block_attention_umma.cu) and on mma.sync (block_attention_tc.cu); IERT_BAD_ARGUMENT: not a case of theirs.
int block_attention_umma(const void* qkv, void* out, const IertBatchView* batch, const IertBlockView* view, int heads, float scale, float* scratch,
                         float* weight_out, const float* inv_freq, int rotary_dim, int pairing, float rot_mul, int splits, int groups, int* err,
                         cudaStream_t stream);
int block_attention_tc(const void* qkv, void* out, const IertBatchView* batch, const IertBlockView* view, int heads, float scale, float* scratch,
                       float* weight_out, const float* inv_freq, int rotary_dim, int pairing, float rot_mul, int splits, int* err, cudaStream_t stream);

namespace iert {

constexpr int BLK = 16;                        // positions of a block
// The smallest scale: the smallest normal fp32 number, so that x / scale is never a division by zero or by a number that has lost digits.
constexpr float MIN_SCALE = 1.17549435e-38f;

// Page `pg` of a sequence (-1, and the error bit, where the table has none or the sequence is longer than its table row).
__device__ __forceinline__ int block_page(const IertBlockView& c, int slot, int pg, int* err) {
  int page = -1;
  if (c.ring_pages < c.table_width || pg < c.table_width) page = c.page_table[(size_t)slot * c.table_width + (pg < c.ring_pages ? pg : pg % c.ring_pages)];
  if (page < 0 || page >= c.n_pages) {
    atomicOr(err, IERT_ERR_PAGE_RANGE);
    return -1;
  }
  return page;
}

// The slot of sequence s, -1 for a padding sequence and (with the error bit) for a slot that the cache does not have.
__device__ __forceinline__ int block_slot(const IertBlockView& c, const IertBatchView& b, int s, int* err) {
  const int slot = s >= 0 ? b.slot_ids[s] : -1;
  if (slot >= c.n_slots) {
    atomicOr(err, IERT_ERR_PAGE_RANGE);
    return -1;
  }
  return slot;
}

// Does a sequence's row of the table reach position `pos`?  (A ring reaches every position.)  If not, the error bit is set.
__device__ __forceinline__ bool block_reaches(const IertBlockView& c, int pos, int* err) {
  if (pos >= 0 && (c.ring_pages < c.table_width || pos / c.page_tokens < c.table_width)) return true;
  atomicOr(err, IERT_ERR_PAGE_RANGE);
  return false;
}

// Which sequence the blocks of threads of grid index `rank` take: the rank-th longest (of equal ones the first), so that those that take long
// do not begin last.  For a step of more blocks than the device holds at once; the whole block of threads calls it, `len` is room for
// ORDERED numbers and one more in shared memory.  With more sequences than that: the rank-th.
constexpr int ORDERED = 256;
__device__ __forceinline__ int rank_th_longest(const IertBatchView& b, int rank, int* len) {
  if (b.n_seqs > ORDERED) return rank;
  for (int i = threadIdx.x; i < b.n_seqs; i += blockDim.x) len[i] = b.slot_ids[i] < 0 ? -1 : b.pos0[i];
  __syncthreads();
  for (int i = threadIdx.x; i < b.n_seqs; i += blockDim.x) {
    const int mine = len[i];
    int longer = 0;
    for (int j = 0; j < b.n_seqs; ++j) longer += len[j] > mine || (len[j] == mine && j < i);
    if (longer == rank) len[ORDERED] = i;
  }
  __syncthreads();
  const int s = len[ORDERED];
  __syncthreads();
  return s;
}

template <int FMT> __device__ __forceinline__ float level_top() { return FMT == IERT_LEVEL_INT8 ? 127.f : 448.f; }

// max |x| over a block from the largest bit pattern of |x|: a NaN is larger than every number, so that it reaches the scale
// and with it everything that reads the block.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Correctly rounded divisions: the levels are then a function of the numbers alone, the same on any machine.
template <int FMT> __device__ __forceinline__ float block_scale(uint32_t largest) {
  const float s = __fdiv_rn(__uint_as_float(largest), level_top<FMT>());
  return s < MIN_SCALE ? MIN_SCALE : s;
}
template <int FMT> __device__ __forceinline__ uint8_t to_level(float x, float scale) {
  const float q = fminf(fmaxf(__fdiv_rn(x, scale), -level_top<FMT>()), level_top<FMT>());
  if (FMT == IERT_LEVEL_INT8) return (uint8_t)(int8_t)__float2int_rn(q);
  return (uint8_t)__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
}
// Levels of four numbers, the first in the lowest byte, to the bit what `to_level` gives, at a fifth of its instructions: x / scale, rounded,
// lies within three roundings of q = x * (1 / scale), so where q (1 - 2^-21) and q (1 + 2^-21) have the same level it is that one, and
// only where a border lies between them (int8: 3 of 100,000 normal numbers, at most 12) is the division carried out.  `inv`: see below.
template <int FMT> __device__ __forceinline__ uint32_t to_levels4(const float* x, float scale, float inv) {
  constexpr float DOWN = 1.f - 0x1p-21f, UP = 1.f + 0x1p-21f;
  uint32_t w[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    float q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = __fmul_rn(__fmul_rn(x[e], inv), side ? UP : DOWN);
    if (FMT == IERT_LEVEL_INT8) {                        // 1.5 * 2^23 more: the nearest whole number (ties to even) stands in the lowest bits
      uint32_t t[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = __float_as_uint(__fadd_rn(q[e], 12582912.f));
      w[side] = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
    } else {
      const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
      w[side] = a | (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3) << 16;
    }
  }
  if (w[0] != w[1] || inv == 0.f) {
    w[0] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[0] |= (uint32_t)to_level<FMT>(x[e], scale) << (8 * e);
  }
  return w[0];
}
// 1 / scale; 0 where it has not all its bits, or the block holds something that is not a finite number.
__device__ __forceinline__ float inverse_of_scale(float scale) { return scale <= 0x1p125f ? __frcp_rn(scale) : 0.f; }
template <int FMT> __device__ __forceinline__ float from_level(uint8_t q) {
  if (FMT == IERT_LEVEL_INT8) return (float)(int8_t)q;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
}

// Largest of a value over a block of threads whose count is a multiple of 32; `red`: one word per warp of shared memory.
__device__ __forceinline__ uint32_t block_max_bits(uint32_t v, uint32_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v = max(v, red[w]);
  return v;
}

// The whole block of threads turns the 16 rows of a tail into levels and their scale.
template <int FMT, typename T>
__device__ void finish_block(const T* tail, int hd, uint8_t* levels, float* scale, uint32_t* red) {
  uint32_t largest = 0;
  for (int i = threadIdx.x; i < BLK * hd; i += blockDim.x) largest = max(largest, abs_bits(to_f32(tail[i])));
  const float s = block_scale<FMT>(block_max_bits(largest, red));
  for (int i = threadIdx.x; i < BLK * hd; i += blockDim.x) levels[i] = to_level<FMT>(to_f32(tail[i]), s);
  if (threadIdx.x == 0) *scale = s;
}

// How many clusters of `size` CTAs the device holds at once of a kernel whose attributes are set (asked once; fewer than its SMs suggest, for a
// cluster stays inside a group of SMs).  `known`: the kernel's own, zeros at first; sizes 1, 2, 4, 8, 16.
template <typename Kernel>
inline int clusters_at_once(Kernel kernel, int size, int threads, size_t smem, int* known) {
  int i = 0;
  while (1 << i < size) ++i;
  if (!known[i]) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1024 * size);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = 1;
    }
    known[i] = n;
  }
  return known[i];
}

}  // namespace iert
