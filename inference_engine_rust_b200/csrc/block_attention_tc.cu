// One-token attention over the 8-bit cache (block_cache.cuh) on the tensor cores, head sizes 64 and 128.
//
// The sequences' keys and values in 8 bits are all that has to come from memory, so everything is arranged around that stream:
//   * A cluster of up to 16 CTAs shares one (sequence, kv head): each takes a run of its blocks, and each adds up a share of the
//     outputs from what the others have put into its shared memory.  One launch, no scratch memory for partial outputs.
//     (Two CTAs of eight warps an SM; in fours, two to a pair, 64 sequences of 4,096 positions took as long in bfloat16 runs and an eighth longer in
//     float32 runs.)
//   * A warp owns a block (16 positions) at a time, with a ring of its own that cp.async fills: no barrier inside the loop.
//   * Levels become fp16 in registers, exactly (int8: 1024 + (q + 128) by a byte permutation, minus 1152; e4m3: a conversion
//     instruction), and are the 16-row operand of mma.m16n8k16: S^T = K Q^T has 16 positions x 8 heads, O^T = V^T P^T 16 dimensions x 8
//     heads, so that a group of up to 8 query heads fills the narrow side.  Queries are scaled by a power of two of their row; bf16
//     numbers are then exact in fp16, fp32 numbers go in twice, the upper 11 bits and the next 11 (`LO`).  Probabilities go in twice in
//     every run: one half alone is off by 2^-12, which moves bfloat16 outputs past the border of their own rounding (64 sequences of up to 4,096
//     positions, e4m3, took 62.0 us so, 64.6 with both).
//   * The order of dimensions inside a product is free as long as both operands agree: a lane takes 16 neighbouring bytes of a key
//     row for four steps (one 16-byte load), and 16 (8) neighbouring dimensions of four value rows.  P^T gets into operand form by
//     two 8 x 8 transpositions in registers (movmatrix).
//   * A block's key scale multiplies its scores, its value scale its probabilities: no level is ever multiplied.  The products of probability and value scale
//     are written as fp16 numbers in a unit, a power of two, that a warp keeps per head and that goes by these products alone: a block of large
//     values that has no weight takes no digits from the others.  It moves where a block's heaviest product leaves [P_LEAST, 2^15], the softmax reference where a
//     score passes it by 2^6, so most blocks cost no maximum across lanes.
// The unfinished block, up to 16 rows in the run's type, is done in fp32 by the last CTA of the cluster, which also stores
// the step's own key and value and turns the block into levels when it is full.
#include <cooperative_groups.h>

#include <utility>

#include "block_cache.cuh"

namespace cg = cooperative_groups;
using namespace iert;

namespace {

constexpr int NSTAGE = 2, GH = 8, MAX_SPLITS = 16, WARPS = 8;
constexpr float HEADROOM = 6.f;           // probabilities stay below 2^6: their product with the largest scale there is still has a number
// A block's heaviest product in its unit: where the unit moves, in [2^(P_TOP - 1), 2^(P_TOP + 1)); then below 2^15 (fp16's largest is just under 2^16) and at
// least P_LEAST.  In two halves a product is off by at most 2^-23 of itself or half of fp16's smallest step, 2^-25: of a block's heaviest 2^-21 in
// bfloat16 runs, 2^-25 in float32 runs.
template <typename T> constexpr int P_TOP = sizeof(T) == 4 ? 8 : 5;
constexpr float P_MOST = 0x1p15f;
template <typename T> constexpr float P_LEAST = sizeof(T) == 4 ? 1.f : 0x1p-4f;
// The output's sums stand in the same unit, so it comes down by no more than this from its highest (the products left out then are below 2^-80 of the heaviest).
constexpr float DOWN = 0x1p40f;
constexpr int TAIL_BLOCKS = 8;            // finished blocks that cost a CTA about as much time as the unfinished one

struct BlockTcParams {
  const void* qkv;
  void* out;
  float* part;                 // [T][kv_heads][slices of 8 heads][blocks][8]: base-2 logarithm of a block's unnormalised weight
  float* weight_out;
  int heads, blocks;
  int by_length;               // longest sequences first
  float scale_log2e;
  const float* inv_freq;
  int rope, rotary_dim, pairing;
  float rot_mul;
  int* err;
};

__device__ __forceinline__ void cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four levels (the bytes of a word) as two pairs of fp16 numbers.
template <int FMT> __device__ __forceinline__ void levels4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (FMT == IERT_LEVEL_INT8) {
    const uint32_t u = w ^ 0x80808080u;                                    // q + 128
    const __half2 off = __float2half2_rn(1152.f);
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);   // 1024 + u in each half
    __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<uint32_t*>(&x);
    hi = *reinterpret_cast<uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}

__device__ __forceinline__ uint32_t half2_bits(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What is left of two numbers when their fp16 roundings are taken away.
__device__ __forceinline__ uint32_t rest_bits(float x, float y, uint32_t hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return half2_bits(x - f.x, y - f.y);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// 16-byte chunk `c` of a block's keys (values) in shared memory, moved inside its 128-byte line so that the loads of a warp, which take
// eight rows of keys or every second row of values at once, meet 32 different banks.
template <int HD> __device__ __forceinline__ int k_chunk(int c) { return HD == 128 ? c ^ (((c >> 3) & 1) << 2) : c; }
template <int HD> __device__ __forceinline__ int v_chunk(int c) { return HD == 128 ? c ^ (((c >> 4) & 3) << 1) : c ^ (((c >> 3) & 3) << 1); }

template <int HD, typename T> struct Shared {
  uint8_t ring[WARPS][NSTAGE][2][BLK * HD];        // (later each warp's partial output, [GH][HD] fp32, in its own ring)
  T tail[2][BLK][HD];
  float q[GH][HD + 4];
  float cs[HD];
  float tail_s[BLK][GH];
  float tail_o[GH][HD];
  float ml[WARPS + 1][GH][2];                      // maximum and sum of each warp, and of the unfinished block
  float o_in[GH * HD + MAX_SPLITS];                // this CTA's share of the outputs, from every CTA of the cluster
  float ml_in[MAX_SPLITS][GH][2];
  float wfac[WARPS + 1][GH];                       // what each warp's sums count for in the CTA's
  float fac[MAX_SPLITS][GH];                       // what each CTA's sums count for in the outputs
  float lse[GH][2];                                // over the cluster: maximum, 1 / sum
  uint32_t red[WARPS];
};

// Element d of a head in fp32, rotated (and then rounded to the run's type, as rotated numbers are everywhere) if the kernel has to.
template <typename T>
__device__ __forceinline__ float head_value(const T* src, int d, const BlockTcParams& p, const float* cs) {
  const float x = to_f32(src[d]);
  if (!p.rope || d >= p.rotary_dim) return x;
  const int half = p.rotary_dim / 2;
  const bool second = p.pairing == IERT_PAIR_HALF ? d >= half : d & 1;
  const int k = p.pairing == IERT_PAIR_HALF ? (second ? d - half : d) : d >> 1;
  const float y = to_f32(src[p.pairing == IERT_PAIR_HALF ? (second ? d - half : d + half) : d ^ 1]);
  return to_f32(from_f32<T>(second ? y * cs[half + k] + x * cs[k] : x * cs[k] - y * cs[half + k]));
}

template <int HD, int FMT, typename T>
__global__ void __launch_bounds__(WARPS * 32, 2) block_attention_tc_kernel(BlockTcParams p, IertBatchView b, IertBlockView c) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  using Sh = Shared<HD, T>;
  constexpr int THREADS = WARPS * 32;
  static_assert(NSTAGE * 2 * BLK >= GH * 4, "a warp's partial output fits in its ring");
  static_assert(THREADS >= MAX_SPLITS * GH && THREADS >= BLK * GH, "a thread per (CTA, head) and per (row, head)");
  Sh& sm = *reinterpret_cast<Sh*>(smem_raw);
  constexpr bool LO = sizeof(T) == 4;              // both halves of queries
  constexpr int KSTEPS = HD / 16, DPL = HD / 8;    // dimensions of a value row that a lane group takes
  cg::cluster_group cluster = cg::this_cluster();
  const int S = gridDim.x, rank = blockIdx.x;      // the cluster is the grid's first axis
  pdl_launch_dependents();
  const int kvh = blockIdx.y, t = p.by_length ? rank_th_longest(b, blockIdx.z, reinterpret_cast<int*>(smem_raw)) : blockIdx.z, group = p.heads / c.kv_heads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
  const int s = sequence_of_token(b, t);
  int slot = block_slot(c, b, s, p.err);
  if (slot >= 0 && !block_reaches(c, b.pos0[s], p.err)) slot = -1;
  pdl_wait();
  T* out = (T*)p.out + ((size_t)t * p.heads + (size_t)kvh * group) * HD;
  if (slot < 0) {                                  // (the same for the whole cluster)
    if (rank == 0)
      for (int i = tid; i < group * HD; i += THREADS) out[i] = from_f32<T>(0.f);
    return;
  }
  cg::cluster_group::arrival_token started = cluster.barrier_arrive();
  const int pos = b.pos0[s], nb = pos / BLK, base = nb * BLK, per_page = c.page_tokens / BLK;
  const int j_min = iert_first_visible(pos, c.window, 0), b_lo = min(j_min / BLK, nb);
  const int per = (nb - b_lo + (S > 1 ? TAIL_BLOCKS : 0) + S - 1) / S;
  const int lo = min(nb, b_lo + rank * per), hi = min(nb, lo + per);
  const int n_mine = max(0, (hi - lo - warp + WARPS - 1) / WARPS);        // blocks lo + warp, lo + warp + WARPS, ...
  const bool owner = rank == S - 1;                // of the unfinished block
  const T* row = (const T*)p.qkv + (size_t)t * (size_t)(p.heads + 2 * c.kv_heads) * HD;

  // Page and scales of 32 of the warp's blocks at a time, one per lane; the groups of even number stand in at[0], the odd ones in at[1].
  int at[2] = {-1, -1};
  float ks[2] = {0.f, 0.f}, vs[2] = {0.f, 0.f};
  auto look_up = [&](int i0, int w) {
    const int x = lo + warp + WARPS * (i0 + lane);
    at[w] = -1; ks[w] = 0.f; vs[w] = 0.f;
    if (i0 + lane < n_mine) {
      const int page = block_page(c, slot, x / per_page, p.err);
      if (page >= 0) {
        at[w] = (page * c.kv_heads + kvh) * per_page + x % per_page;
        ks[w] = c.k_scale[at[w]];
        vs[w] = c.v_scale[at[w]];
      }
    }
  };
  auto issue = [&](int i) {
    if (i < n_mine) {
      const int a = __shfl_sync(0xffffffffu, (i >> 5) & 1 ? at[1] : at[0], i & 31);
      if (a >= 0) {
        uint8_t *kd = sm.ring[warp][i % NSTAGE][0], *vd = sm.ring[warp][i % NSTAGE][1];
        const uint8_t *kq = (const uint8_t*)c.k + (size_t)a * (BLK * HD), *vq = (const uint8_t*)c.v + (size_t)a * (BLK * HD);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          cp16(kd + k_chunk<HD>(lane + 32 * j) * 16, kq + (lane + 32 * j) * 16);
          cp16(vd + v_chunk<HD>(lane + 32 * j) * 16, vq + (lane + 32 * j) * 16);
        }
      }
    }
    cp_commit();
  };

  for (int g0 = 0; g0 < group; g0 += GH) {
    const int n_g = min(GH, group - g0), head0 = kvh * group + g0;
    float* part = c.weight ? p.part + (((size_t)t * c.kv_heads + kvh) * ((group + GH - 1) / GH) + g0 / GH) * p.blocks * GH : nullptr;
    look_up(0, 0);
    look_up(32, 1);
#pragma unroll
    for (int i = 0; i < NSTAGE - 1; ++i) issue(i);

    // ---- queries and, with the unfinished block's owner, its rows
    if (g0 == 0) {
      if (p.rope) {
        const float where = (float)(pos + (c.shift ? c.shift[slot] : 0));
        for (int k = tid; k < p.rotary_dim / 2; k += THREADS) {
          float sn, co;
          sincosf(where * p.inv_freq[k], &sn, &co);
          sm.cs[k] = co * p.rot_mul;
          sm.cs[p.rotary_dim / 2 + k] = sn * p.rot_mul;
        }
        __syncthreads();
      }
      if (owner) {
        const size_t off = ((size_t)slot * c.kv_heads + kvh) * BLK * HD;
        T *tk = (T*)c.tail_k + off, *tv = (T*)c.tail_v + off;
        const int old = (pos - base) * HD;
        constexpr int V = 16 / sizeof(T);
#pragma unroll 4
        for (int i = tid * V; i < old; i += THREADS * V) {
          const uint4 x = *reinterpret_cast<const uint4*>(tk + i), y = *reinterpret_cast<const uint4*>(tv + i);
          *reinterpret_cast<uint4*>(&sm.tail[0][0][0] + i) = x;
          *reinterpret_cast<uint4*>(&sm.tail[1][0][0] + i) = y;
        }
        const T *kn = row + (size_t)(p.heads + kvh) * HD, *vn = row + (size_t)(p.heads + c.kv_heads + kvh) * HD;
        for (int d = tid; d < HD; d += THREADS) {
          const T x = from_f32<T>(head_value(kn, d, p, sm.cs)), v = vn[d];
          sm.tail[0][pos - base][d] = x;
          sm.tail[1][pos - base][d] = v;
          tk[old + d] = x;
          tv[old + d] = v;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < GH * HD / THREADS; ++i) {
      const int r = (tid + i * THREADS) / HD, d = (tid + i * THREADS) % HD;
      sm.q[r][d] = r < n_g ? head_value(row + (size_t)(head0 + r) * HD, d, p, sm.cs) : 0.f;
    }
    __syncthreads();

    // ---- the narrow operand of the scores: head g, scaled by a power of two so that its largest number lies in [2^13, 2^14)
    float rs[2];                                   // what makes scores of the products, heads 2 tq and 2 tq + 1
    uint32_t qh[KSTEPS][2], ql[LO ? KSTEPS : 1][2];
    {
      uint32_t largest = 0;
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j) {
        const float4 x = *reinterpret_cast<const float4*>(&sm.q[g][64 * (j >> 2) + 16 * tq + 4 * (j & 3)]);
        largest = max(max(largest, max(abs_bits(x.x), abs_bits(x.y))), max(abs_bits(x.z), abs_bits(x.w)));
      }
      largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
      largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
      const int e = min(max((int)(largest >> 23), 14), 253);
      const float f = __uint_as_float((uint32_t)(267 - e) << 23), back = __uint_as_float((uint32_t)(e - 13) << 23) * p.scale_log2e;
      rs[0] = __shfl_sync(0xffffffffu, back, 8 * tq);
      rs[1] = __shfl_sync(0xffffffffu, back, 8 * tq + 4);
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j) {
        const float4 x = *reinterpret_cast<const float4*>(&sm.q[g][64 * (j >> 2) + 16 * tq + 4 * (j & 3)]);
        qh[j][0] = half2_bits(x.x * f, x.y * f);
        qh[j][1] = half2_bits(x.z * f, x.w * f);
        if (LO) {
          ql[j][0] = rest_bits(x.x * f, x.y * f, qh[j][0]);
          ql[j][1] = rest_bits(x.z * f, x.w * f, qh[j][1]);
        }
      }
    }

    // ---- the unfinished block, in fp32: a thread per (row, head), then per dimension
    if (owner) {
      const int r = tid >> 3, h = tid & 7;           // (threads beyond the 16 rows have nothing to do)
      float sc = -INFINITY;
      if (r < BLK && base + r <= pos && base + r >= j_min) {
        float dot = 0.f;
#pragma unroll 8
        for (int d = 0; d < HD; d += 4) {
          const float4 x = *reinterpret_cast<const float4*>(&sm.q[h][d]);
          const T* k = &sm.tail[0][r][d];
          dot = fmaf(x.x, to_f32(k[0]), dot); dot = fmaf(x.y, to_f32(k[1]), dot);
          dot = fmaf(x.z, to_f32(k[2]), dot); dot = fmaf(x.w, to_f32(k[3]), dot);
        }
        sc = dot * p.scale_log2e;
      }
      if (r < BLK) sm.tail_s[r][h] = sc;
      __syncthreads();
      float mx = -INFINITY, l = 0.f;
#pragma unroll
      for (int i = 0; i < BLK; ++i) mx = fmaxf(mx, sm.tail_s[i][h]);
      const float pr = mx == -INFINITY ? (sc == sc ? 0.f : sc) : ex2(sc - mx);
      __syncthreads();
      if (r < BLK) sm.tail_s[r][h] = pr;
      __syncthreads();
      if (r == 0) {
#pragma unroll
        for (int i = 0; i < BLK; ++i) l += sm.tail_s[i][h];
        sm.ml[WARPS][h][0] = mx;
        sm.ml[WARPS][h][1] = l;
        if (part) part[(size_t)nb * GH + h] = mx + log2f(l);
      }
      constexpr int PER = GH * HD / THREADS < 1 ? 1 : GH * HD / THREADS;     // heads of a thread
      for (int e = tid; e < HD * GH / PER; e += THREADS) {
        const int d = e % HD, k0 = e / HD * PER;
        float acc[PER] = {};
        for (int i = max(0, j_min - base); i <= pos - base; ++i) {
          const float v = to_f32(sm.tail[1][i][d]);
#pragma unroll
          for (int k = 0; k < PER; ++k) acc[k] = fmaf(sm.tail_s[i][k0 + k], v, acc[k]);
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) sm.tail_o[k0 + k][d] = acc[k];
      }
    }

    // ---- the finished blocks.  o[i]: dimensions DPL g + 2 i (0, 1) and + 1 (2, 3), heads 2 tq (0, 2) and 2 tq + 1 (1, 3)
    float o[DPL / 2][4];
#pragma unroll
    for (int n = 0; n < DPL / 2; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};      // probabilities are relative to 2^ref
    float root[2] = {0.f, 0.f}, least[2] = {INFINITY, INFINITY};   // o's unit is root^-2 (0: none yet); the smallest root so far
    for (int i = 0; i < n_mine; ++i) {
      if ((i & 31) == 0 && i > 0) {                 // the next 32 blocks
        if ((i >> 5) & 1) look_up(i + 32, 0); else look_up(i + 32, 1);
      }
      issue(i + NSTAGE - 1);
      const bool odd = (i >> 5) & 1;
      const int a = __shfl_sync(0xffffffffu, odd ? at[1] : at[0], i & 31);
      const float k_scale = __shfl_sync(0xffffffffu, odd ? ks[1] : ks[0], i & 31), v_scale = __shfl_sync(0xffffffffu, odd ? vs[1] : vs[0], i & 31);
      const int x = lo + warp + WARPS * i;
      cp_wait<NSTAGE - 1>();
      __syncwarp();
      if (a < 0) {                                   // a page that the pool does not have: the block counts for nothing
        if (part && lane < GH) part[(size_t)x * GH + lane] = -INFINITY;
        continue;
      }
      const uint8_t *kt = sm.ring[warp][i % NSTAGE][0], *vt = sm.ring[warp][i % NSTAGE][1];
      float sc[4] = {0.f, 0.f, 0.f, 0.f}, sl[4] = {0.f, 0.f, 0.f, 0.f};      // positions g (0, 1) and g + 8 (2, 3), heads as above
#pragma unroll
      for (int j = 0; j < HD / 64; ++j) {
        const uint4 w0 = *reinterpret_cast<const uint4*>(kt + k_chunk<HD>(g * (HD / 16) + 4 * j + tq) * 16);
        const uint4 w1 = *reinterpret_cast<const uint4*>(kt + k_chunk<HD>((g + 8) * (HD / 16) + 4 * j + tq) * 16);
        const uint32_t wa[4] = {w0.x, w0.y, w0.z, w0.w}, wb[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t f[4];
          levels4<FMT>(wa[e], f[0], f[2]);
          levels4<FMT>(wb[e], f[1], f[3]);
          // two sums of half the dimensions each (float runs: upper and lower halves of the queries), so that products wait for one another less
          if (LO) {
            mma_f16(sc, f, qh[4 * j + e][0], qh[4 * j + e][1]);
            mma_f16(sl, f, ql[4 * j + e][0], ql[4 * j + e][1]);
          } else {
            mma_f16(e & 1 ? sl : sc, f, qh[4 * j + e][0], qh[4 * j + e][1]);
          }
        }
      }
      float v[4], y[4];
      bool far = false;
      const int first = j_min - x * BLK;             // positions below are outside the window
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = (sc[e] + sl[e]) * (k_scale * rs[e & 1]);
        if (first > 0 && g + 8 * (e >> 1) < first) v[e] = -INFINITY;
        y[e] = v[e] - ref[e & 1];
        far |= !(y[e] <= HEADROOM);
      }
      if (__any_sync(0xffffffffu, far)) {            // the first block, a score far above what came before, or something that is not a number
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(v[h], v[h + 2]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
          const float to = fmaxf(ref[h], mx);
          const float alpha = to == ref[h] ? 1.f : ex2(ref[h] - to);
          ref[h] = to;
          l[h] *= alpha;
#pragma unroll
          for (int n = 0; n < DPL / 2; ++n) { o[n][h] *= alpha; o[n][h + 2] *= alpha; }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = v[e] == -INFINITY ? v[e] : v[e] - ref[e & 1];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = ex2(y[e]);
      const float s0 = y[0] + y[2], s1 = y[1] + y[3];
      l[0] += s0;
      l[1] += s1;
      float w[4];
      bool large = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = y[e] * v_scale * root[e & 1] * root[e & 1];
        large |= !(w[e] <= P_MOST);
      }
      // lanes 4 g + tq: has any g a product of head 2 tq (2 tq + 1) that is not too small?
      uint32_t some0 = __ballot_sync(0xffffffffu, fmaxf(w[0], w[2]) >= P_LEAST<T>), some1 = __ballot_sync(0xffffffffu, fmaxf(w[1], w[3]) >= P_LEAST<T>);
      some0 |= some0 >> 16; some1 |= some1 >> 16;
      some0 |= some0 >> 8; some1 |= some1 >> 8;
      some0 |= some0 >> 4; some1 |= some1 >> 4;
      if (__any_sync(0xffffffffu, large) || (some0 & some1 & 0xfu) != 0xfu) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(y[h] * v_scale, y[h + 2] * v_scale);
#pragma unroll
          for (int x2 = 4; x2 < 32; x2 <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x2));
          if (mx > 0.f) {                            // (a block without any leaves the unit as it is)
            const int e = (int)(__float_as_uint(mx) >> 23);
            const float to = fminf(__uint_as_float((uint32_t)(((P_TOP<T> + 127 - max(e, 1)) >> 1) + 127) << 23), least[h] * DOWN);
            const float f = root[h] > 0.f ? to * __uint_as_float((254u << 23) - __float_as_uint(root[h])) : 0.f;      // to / root
            root[h] = to;
            least[h] = fminf(least[h], to);
#pragma unroll
            for (int n = 0; n < DPL / 2; ++n) { o[n][h] = o[n][h] * f * f; o[n][h + 2] = o[n][h + 2] * f * f; }
          }
          w[h] = y[h] * v_scale * root[h] * root[h];
          w[h + 2] = y[h + 2] * v_scale * root[h] * root[h];
        }
      }
      if (part) {                                    // the block's sums: lanes of g < 4 end with head 2 tq, the others with 2 tq + 1
        float keep = g & 4 ? s1 : s0;
        keep += __shfl_xor_sync(0xffffffffu, g & 4 ? s0 : s1, 16);
        keep += __shfl_xor_sync(0xffffffffu, keep, 8);
        keep += __shfl_xor_sync(0xffffffffu, keep, 4);
        if ((g & 3) == 0) part[(size_t)x * GH + 2 * tq + (g >> 2)] = (g & 4 ? ref[1] : ref[0]) + log2f(keep);
      }
      const uint32_t p0 = half2_bits(w[0], w[1]), p1 = half2_bits(w[2], w[3]);
      const uint32_t b0 = transposed(p0), b1 = transposed(p1);
      const uint32_t r0 = transposed(rest_bits(w[0], w[1], p0)), r1 = transposed(rest_bits(w[2], w[3], p1));
      // values of rows 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9, dimensions [DPL g, DPL (g + 1))
      uint32_t vw[4][DPL / 4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int vr_ = 2 * tq + (r & 1) + 8 * (r >> 1);
        if (HD == 128) {
          const uint4 w4 = *reinterpret_cast<const uint4*>(vt + v_chunk<HD>(vr_ * 8 + g) * 16);
          vw[r][0] = w4.x; vw[r][1] = w4.y; vw[r][DPL / 4 - 2] = w4.z; vw[r][DPL / 4 - 1] = w4.w;
        } else {
          const uint2 w2 = *reinterpret_cast<const uint2*>(vt + v_chunk<HD>(vr_ * 4 + (g >> 1)) * 16 + (g & 1) * 8);
          vw[r][0] = w2.x; vw[r][1] = w2.y;
        }
      }
#pragma unroll
      for (int w = 0; w < DPL / 4; ++w)
#pragma unroll
        for (int z = 0; z < 2; ++z) {                // two dimensions at a time: bytes of two rows side by side
          const uint32_t sel = z ? 0x7362 : 0x5140;
          uint32_t f[4];
          levels4<FMT>(__byte_perm(vw[0][w], vw[1][w], sel), f[0], f[1]);
          levels4<FMT>(__byte_perm(vw[2][w], vw[3][w], sel), f[2], f[3]);
          mma_f16(o[2 * w + z], f, b0, b1);
          mma_f16(o[2 * w + z], f, r0, r1);
        }
      __syncwarp();                                  // the stage may be filled again
    }
    cp_wait<0>();
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], w);
    float* mine = reinterpret_cast<float*>(&sm.ring[warp][0][0][0]);       // [GH][HD]
    const float b0 = __uint_as_float((254u << 23) - __float_as_uint(root[0])), b1 = __uint_as_float((254u << 23) - __float_as_uint(root[1]));      // 1 / root
#pragma unroll
    for (int n = 0; n < DPL / 2; ++n) {
      *reinterpret_cast<float2*>(mine + (2 * tq) * HD + DPL * g + 2 * n) = make_float2(o[n][0] * b0 * b0, o[n][2] * b0 * b0);
      *reinterpret_cast<float2*>(mine + (2 * tq + 1) * HD + DPL * g + 2 * n) = make_float2(o[n][1] * b1 * b1, o[n][3] * b1 * b1);
    }
    if (g == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) { sm.ml[warp][2 * tq + h][0] = ref[h]; sm.ml[warp][2 * tq + h][1] = l[h]; }
    }
    __syncthreads();
    if (tid < (WARPS + 1) * GH) {                  // warps in their order, then the unfinished block
      const int w = tid / GH, h = tid % GH;
      const int n = owner ? WARPS + 1 : WARPS;
      float mm = -INFINITY;
      for (int k = 0; k < n; ++k) mm = fmaxf(mm, sm.ml[k][h][0]);
      sm.wfac[w][h] = w >= n ? 0.f : sm.ml[w][h][0] == mm ? 1.f : ex2(sm.ml[w][h][0] - mm);
    }
    cluster.barrier_wait(std::move(started));      // every CTA runs (and has read what it was sent for the heads before)
    __syncthreads();

    // ---- the CTA's partial result goes to the CTAs that add up its pieces
    const int share = (n_g * HD + S - 1) / S;
#pragma unroll
    for (int k = 0; k < GH * HD / THREADS; ++k) {
      const int i = tid + k * THREADS, h = i / HD, d = i % HD;
      if (i >= n_g * HD) break;
      float acc = owner ? sm.wfac[WARPS][h] * sm.tail_o[h][d] : 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) acc += sm.wfac[w][h] * reinterpret_cast<const float*>(&sm.ring[w][0][0][0])[h * HD + d];
      const int to = i / share;
      cluster.map_shared_rank(&sm.o_in[0], to)[rank * share + i - to * share] = acc;
    }
    if (tid < S * GH) {
      const int to = tid / GH, h = tid % GH, n = owner ? WARPS + 1 : WARPS;
      float mm = -INFINITY, ll = 0.f;
      for (int k = 0; k < n; ++k) { mm = fmaxf(mm, sm.ml[k][h][0]); ll += sm.wfac[k][h] * sm.ml[k][h][1]; }
      *reinterpret_cast<float2*>(cluster.map_shared_rank(&sm.ml_in[rank][h][0], to)) = make_float2(mm, ll);
    }
    cluster.sync();

    // ---- this CTA's share of the outputs
    if (tid < S * GH) {
      const int r = tid / GH, h = tid % GH;
      float mm = -INFINITY, ll = 0.f;
      for (int k = 0; k < S; ++k) mm = fmaxf(mm, sm.ml_in[k][h][0]);
      for (int k = 0; k < S; ++k) ll += (sm.ml_in[k][h][0] == mm ? 1.f : ex2(sm.ml_in[k][h][0] - mm)) * sm.ml_in[k][h][1];
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      sm.fac[r][h] = (sm.ml_in[r][h][0] == mm ? 1.f : ex2(sm.ml_in[r][h][0] - mm)) * inv;
      if (r == 0) { sm.lse[h][0] = mm; sm.lse[h][1] = inv; }
    }
    __syncthreads();
    for (int k = tid; k < share; k += THREADS) {
      const int i = rank * share + k;
      if (i >= n_g * HD) break;
      float acc = 0.f;
      for (int r = 0; r < S; ++r) acc += sm.fac[r][i / HD] * sm.o_in[r * share + k];
      out[(size_t)g0 * HD + i] = from_f32<T>(acc);
    }
    if (part) {
      // weight of block x: the sum over the group's heads, in their order, of 2^(part - maximum) / sum
      const int end = owner ? nb + 1 : hi;
      for (int x = lo + tid; x < end; x += THREADS) {
        const int page = block_page(c, slot, x / per_page, p.err);
        if (page < 0) continue;
        const size_t i = ((size_t)page * c.kv_heads + kvh) * per_page + x % per_page;
        float w = g0 > 0 ? p.weight_out[i] : x == nb && pos == base ? 0.f : c.weight[i];
        const float4 a = *reinterpret_cast<const float4*>(part + (size_t)x * GH), b4 = *reinterpret_cast<const float4*>(part + (size_t)x * GH + 4);
        const float e[GH] = {a.x, a.y, a.z, a.w, b4.x, b4.y, b4.z, b4.w};
#pragma unroll
        for (int h = 0; h < GH; ++h)
          if (h < n_g) w += ex2(e[h] - sm.lse[h][0]) * sm.lse[h][1];
        p.weight_out[i] = w;
      }
    }
    if (g0 + GH < group) {
      __syncthreads();
      started = cluster.barrier_arrive();
    }
  }

  if (owner && pos - base == BLK - 1) {              // the block is full: from the next step on it is read in 8 bits
    const int page = block_page(c, slot, nb / per_page, p.err);
    if (page >= 0) {
      const size_t i = ((size_t)page * c.kv_heads + kvh) * per_page + nb % per_page;
      finish_block<FMT>(&sm.tail[0][0][0], HD, (uint8_t*)c.k + i * BLK * HD, c.k_scale + i, sm.red);
      finish_block<FMT>(&sm.tail[1][0][0], HD, (uint8_t*)c.v + i * BLK * HD, c.v_scale + i, sm.red);
    }
  }
}

template <int HD, int FMT, typename T>
int launch(BlockTcParams p, const IertBatchView& b, const IertBlockView& c, int splits, cudaStream_t stream) {
  auto kernel = block_attention_tc_kernel<HD, FMT, T>;
  const size_t smem = sizeof(Shared<HD, T>);
  static bool configured = false;
  static int known[5];
  if (!configured) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return iert_check_launch("block_attention (attributes)");
    configured = true;
  }
  const long long pairs = (long long)c.kv_heads * b.n_seqs;
  const int sms = iert_sm_count_cached();
  if (splits == 0) {
    // The largest clusters that all run at once (8 sequences of 2,048 positions with 8 key heads: 22.8, 17.8, 14.6, 24.0 us with 1, 2, 4, 8 CTAs
    // to a pair; two of 3,000: 19.1 us in clusters of 16, of which the device holds 14, and 12.3 of 8), those of 16 for sequences that may be long
    // (one sequence of 700 positions: 8.1 us, 7.2 in clusters of 8; of 3,000: 9.4 and 9.3; of 6,000: 11.3 and 11.8).  Between one and two pairs an SM a second CTA evens
    // out what the SMs have to do, which is worth its start for long sequences (24 of 4,096: 38.4 us for 50.8, of 1,024: 23.3 for 21.2).
    const long long reach = (long long)c.ring_pages * c.page_tokens;       // the most that a sequence holds
    for (splits = reach >= 4096 ? MAX_SPLITS : 8; splits > 1 && pairs > clusters_at_once(kernel, splits, WARPS * 32, smem, known);) splits >>= 1;
    if (splits == 1 && pairs <= 2LL * sms && reach >= 4096) splits = 2;
  }
  p.by_length = pairs * splits > 2LL * sms;      // (64 sequences of up to 4,096 positions, e4m3: 85 us as they stand, 74 so)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, c.kv_heads, b.n_seqs);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = iert_pdl_enabled ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, p, b, c);
  return iert_check_launch("block_attention");
}

}  // namespace

// `splits` (1, 2, 4, 8, 16): CTAs that share a sequence's kv head; 0: by the rule above.
int block_attention_tc(const void* qkv, void* out, const IertBatchView* batch, const IertBlockView* view, int heads, float scale,
                       float* scratch, float* weight_out, const float* inv_freq, int rotary_dim, int pairing, float rot_mul, int splits,
                       int* err, cudaStream_t stream) {
  const IertBlockView& c = *view;
  if ((c.head_dim != 64 && c.head_dim != 128) || c.kv_heads <= 0 || heads <= 0 || heads % c.kv_heads || batch->n_tokens != batch->n_seqs ||
      batch->n_seqs > 65535 || c.kv_heads > 65535 || c.page_tokens <= 0 || c.page_tokens % BLK || c.table_width <= 0 || c.ring_pages <= 0 ||
      c.ring_pages > c.table_width || c.n_pages <= 0 || c.n_slots <= 0 || c.window < 0 ||
      !scratch || (c.weight && (c.window || !weight_out)) || ((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.tail_k | (uintptr_t)c.tail_v | (uintptr_t)scratch) % 16 ||
      (inv_freq && (rotary_dim < 0 || rotary_dim > c.head_dim || (rotary_dim & 1) || (pairing != IERT_PAIR_HALF && pairing != IERT_PAIR_INTERLEAVED))))
    return IERT_BAD_ARGUMENT;
  if (splits < 0 || splits > MAX_SPLITS || (splits & (splits - 1))) return IERT_BAD_ARGUMENT;
  BlockTcParams p = {};
  p.qkv = qkv; p.out = out; p.part = scratch; p.weight_out = weight_out;
  p.heads = heads; p.blocks = c.table_width * (c.page_tokens / BLK);
  p.scale_log2e = scale * 1.44269504088896340736f;
  p.inv_freq = inv_freq; p.rope = inv_freq != nullptr; p.rotary_dim = rotary_dim; p.pairing = pairing; p.rot_mul = rot_mul; p.err = err;
  const int which = (c.head_dim == 128 ? 4 : 0) + (c.format == IERT_LEVEL_E4M3 ? 2 : 0) + (c.tail_dtype == IERT_BF16 ? 1 : 0);
  switch (which) {
    case 0: return launch<64, IERT_LEVEL_INT8, float>(p, *batch, c, splits, stream);
    case 1: return launch<64, IERT_LEVEL_INT8, __nv_bfloat16>(p, *batch, c, splits, stream);
    case 2: return launch<64, IERT_LEVEL_E4M3, float>(p, *batch, c, splits, stream);
    case 3: return launch<64, IERT_LEVEL_E4M3, __nv_bfloat16>(p, *batch, c, splits, stream);
    case 4: return launch<128, IERT_LEVEL_INT8, float>(p, *batch, c, splits, stream);
    case 5: return launch<128, IERT_LEVEL_INT8, __nv_bfloat16>(p, *batch, c, splits, stream);
    case 6: return launch<128, IERT_LEVEL_E4M3, float>(p, *batch, c, splits, stream);
    default: return launch<128, IERT_LEVEL_E4M3, __nv_bfloat16>(p, *batch, c, splits, stream);
  }
}
