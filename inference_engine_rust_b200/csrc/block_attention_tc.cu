// One-token attention over the 8-bit cache (block_cache.cuh) on the tensor cores, head sizes 64 and 128.
//
// The sequences' keys and values in 8 bits are all that has to come from memory, so everything is arranged around that stream:
//   * A cluster of up to 16 CTAs shares one (sequence, kv head): each takes a run of its blocks, and their partial results meet in
//     one another's shared memory.  One launch, no scratch memory for partial outputs, no second kernel.
//   * A warp owns a block (16 positions) at a time, with a ring of its own that cp.async fills: no barrier inside the loop.
//   * Levels become fp16 in registers, exactly (int8: 1024 + (q + 128) by a byte permutation, minus 1152; e4m3: a conversion
//     instruction), and are operands of mma.m16n8k16 with fp32 sums.  The tile's 16 rows are 8 query heads twice: rows 0-7 the upper
//     11 bits of a query (scaled by a power of two of its row), rows 8-15 the next 11.  Products with a row's both halves are
//     exact to 2^-22, so float32 runs and bfloat16 runs take the same kernel, and weights (which eviction adds up) are as good as fp32.
//     Probabilities go into the second product the same way.  A bf16 group of up to 8 heads leaves half a tile empty anyway.
//   * The order of dimensions inside a product is free as long as both operands agree: a lane takes 16 neighbouring bytes of a key
//     row for four steps (one 16-byte load), and 16 (8) neighbouring dimensions of four value rows.
//   * A block's key scale multiplies its scores, its value scale the 16-position partial product: no level is ever multiplied.
// The unfinished block, fewer than 17 rows in the run's type, is done in fp32 by the last CTA of the cluster, which also stores
// the step's own key and value and turns the block into levels when it is full.
#include <cooperative_groups.h>

#include "block_cache.cuh"

namespace cg = cooperative_groups;
using namespace iert;

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32, NSTAGE = 3, GH = 8;
constexpr float P_SHIFT = 14.f;           // probabilities are at most 2^14 in the second product: fp16 keeps what is 2^-38 of the largest

struct BlockTcParams {
  const void* qkv;
  void* out;
  float* part;                 // [T][heads][blocks]: base-2 logarithm of a block's unnormalised weight
  float* weight_out;
  int heads, blocks;
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

// Two numbers as the upper 11 bits of each and what is left of them, in fp16.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// 16-byte chunk `c` of a block's keys (values) in shared memory, moved inside its 128-byte line so that the loads of a warp, which take
// eight rows of keys or every second row of values at once, meet 32 different banks.
template <int HD> __device__ __forceinline__ int k_chunk(int c) { return HD == 128 ? c ^ (((c >> 3) & 1) << 2) : c; }
template <int HD> __device__ __forceinline__ int v_chunk(int c) { return HD == 128 ? c ^ (((c >> 4) & 3) << 1) : c ^ (((c >> 3) & 3) << 1); }

template <int HD, typename T> struct Shared {
  static constexpr int QS = HD + 4;               // row stride of the queries
  uint8_t ring[WARPS][NSTAGE][2][BLK * HD];        // (later each warp's partial output, [GH][HD] fp32, in its own first stages)
  T tail[2][BLK][HD];
  float q[GH][QS];
  float cs[HD];
  float tail_s[BLK][GH];
  float tail_o[GH][HD];
  float ml[WARPS + 1][GH][2];
  float o[GH][HD];                                 // the CTA's result: read by the whole cluster
  float oml[GH][2];
  float lse[GH][2];                                // over the cluster: maximum, 1 / sum
  uint32_t red[WARPS];
};

template <int HD, int FMT, typename T>
__global__ void __launch_bounds__(THREADS, 3) block_attention_tc_kernel(BlockTcParams p, IertBatchView b, IertBlockView c) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  using Sh = Shared<HD, T>;
  static_assert(NSTAGE * 2 * BLK >= GH * 4, "a warp's partial output fits in its ring");
  Sh& sm = *reinterpret_cast<Sh*>(smem_raw);
  constexpr int KSTEPS = HD / 16, DPL = HD / 8;    // dimensions of a value row that a lane group takes
  cg::cluster_group cluster = cg::this_cluster();
  const int S = gridDim.x, rank = blockIdx.x;      // the cluster is the grid's first axis
  pdl_launch_dependents();
  const int kvh = blockIdx.y, t = blockIdx.z, group = p.heads / c.kv_heads;
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
  const int pos = b.pos0[s], nb = pos / BLK, base = nb * BLK, per_page = c.page_tokens / BLK;
  const int j_min = iert_first_visible(pos, c.window, 0), b_lo = min(j_min / BLK, nb);
  const int per = (nb - b_lo + S - 1) / S;
  const int lo = min(nb, b_lo + rank * per), hi = min(nb, lo + per);
  const int n_mine = max(0, (hi - lo - warp + WARPS - 1) / WARPS);        // blocks lo + warp, lo + warp + WARPS, ...
  const bool owner = rank == S - 1;                // of the unfinished block
  const T* row = (const T*)p.qkv + (size_t)t * (size_t)(p.heads + 2 * c.kv_heads) * HD;

  // Page and scales of 32 of the warp's blocks at a time, one per lane.
  int at = -1, at_next = -1;
  float ks = 0.f, vs = 0.f, ks_next = 0.f, vs_next = 0.f;
  auto look_up = [&](int i0, int& a, float& k, float& v) {
    const int x = lo + warp + WARPS * (i0 + lane);
    a = -1; k = 0.f; v = 0.f;
    if (i0 + lane < n_mine) {
      const int page = block_page(c, slot, x / per_page, p.err);
      if (page >= 0) {
        a = (page * c.kv_heads + kvh) * per_page + x % per_page;
        k = c.k_scale[a];
        v = c.v_scale[a];
      }
    }
  };
  auto issue = [&](int i) {                        // (i & 31 of the group that `at` or `at_next` holds)
    if (i < n_mine) {
      const int a = __shfl_sync(0xffffffffu, ((i >> 5) & 1) == 0 ? at : at_next, i & 31);
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
    look_up(0, at, ks, vs);
    look_up(32, at_next, ks_next, vs_next);
#pragma unroll
    for (int i = 0; i < NSTAGE - 1; ++i) issue(i);

    // ---- queries (and, with the unfinished block's owner, its rows), rotated if the kernel has to
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
        for (int i = tid; i < old; i += THREADS) { (&sm.tail[0][0][0])[i] = tk[i]; (&sm.tail[1][0][0])[i] = tv[i]; }
        const T *kn = row + (size_t)(p.heads + kvh) * HD, *vn = row + (size_t)(p.heads + c.kv_heads + kvh) * HD;
        for (int d = tid; d < HD; d += THREADS) {
          T x = kn[d];
          if (p.rope) {
            const int half = p.rotary_dim / 2;
            const bool second = p.pairing == IERT_PAIR_HALF ? d >= half : d & 1;
            if (d < p.rotary_dim) {
              const int k = p.pairing == IERT_PAIR_HALF ? (second ? d - half : d) : d >> 1;
              const float y = to_f32(kn[p.pairing == IERT_PAIR_HALF ? (second ? d - half : d + half) : d ^ 1]), f = to_f32(x);
              x = from_f32<T>(second ? y * sm.cs[half + k] + f * sm.cs[k] : f * sm.cs[k] - y * sm.cs[half + k]);
            }
          }
          const T v = vn[d];
          sm.tail[0][pos - base][d] = x;
          sm.tail[1][pos - base][d] = v;
          tk[old + d] = x;
          tv[old + d] = v;
        }
      }
    }
    for (int i = tid; i < GH * HD; i += THREADS) {
      const int r = i / HD, d = i % HD;
      float x = 0.f;
      if (r < n_g) {
        const T* q = row + (size_t)(head0 + r) * HD;
        x = to_f32(q[d]);
        if (p.rope && d < p.rotary_dim) {
          const int half = p.rotary_dim / 2;
          const bool second = p.pairing == IERT_PAIR_HALF ? d >= half : d & 1;
          const int k = p.pairing == IERT_PAIR_HALF ? (second ? d - half : d) : d >> 1;
          const float y = to_f32(q[p.pairing == IERT_PAIR_HALF ? (second ? d - half : d + half) : d ^ 1]);
          x = second ? y * sm.cs[half + k] + x * sm.cs[k] : x * sm.cs[k] - y * sm.cs[half + k];
        }
      }
      sm.q[r][d] = x;
    }
    __syncthreads();

    // ---- query fragments: row g (head g), scaled by a power of two to [1, 4), in two halves
    float row_scale;
    uint32_t qf[KSTEPS][4];
    {
      uint32_t largest = 0;
#pragma unroll
      for (int j = 0; j < HD / 64; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(&sm.q[g][64 * j + 16 * tq + 4 * w]);
          largest = max(max(largest, max(abs_bits(x.x), abs_bits(x.y))), max(abs_bits(x.z), abs_bits(x.w)));
        }
      largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
      largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
      const int e = min(max((int)(largest >> 23), 1), 253);              // exponent of the row's largest number
      const float f = __uint_as_float((uint32_t)(254 - e) << 23);
      row_scale = __uint_as_float((uint32_t)e << 23) * p.scale_log2e;
#pragma unroll
      for (int j = 0; j < HD / 64; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(&sm.q[g][64 * j + 16 * tq + 4 * w]);
          split2(x.x * f, x.y * f, qf[4 * j + w][0], qf[4 * j + w][1]);
          split2(x.z * f, x.w * f, qf[4 * j + w][2], qf[4 * j + w][3]);
        }
    }

    // ---- the unfinished block, in fp32: a thread per (row, head), then per dimension
    if (owner) {
      const int r = tid >> 3, h = tid & 7;
      if (tid < BLK * GH) {
        float dot = 0.f;
        if (base + r <= pos) {
#pragma unroll 8
          for (int d = 0; d < HD; d += 4) {
            const float4 x = *reinterpret_cast<const float4*>(&sm.q[h][d]);
            const T* k = &sm.tail[0][r][d];
            dot = fmaf(x.x, to_f32(k[0]), dot); dot = fmaf(x.y, to_f32(k[1]), dot);
            dot = fmaf(x.z, to_f32(k[2]), dot); dot = fmaf(x.w, to_f32(k[3]), dot);
          }
        }
        sm.tail_s[r][h] = base + r <= pos && base + r >= j_min ? dot * p.scale_log2e : -INFINITY;
      }
      __syncthreads();
      if (tid < GH) {
        float mx = -INFINITY, l = 0.f;
        for (int i = 0; i < BLK; ++i) mx = fmaxf(mx, sm.tail_s[i][tid]);
        for (int i = 0; i < BLK; ++i) {
          const float x = sm.tail_s[i][tid];
          const float pr = mx == -INFINITY ? (x == x ? 0.f : x) : exp2f(x - mx);
          sm.tail_s[i][tid] = pr;
          l += pr;
        }
        sm.ml[WARPS][tid][0] = mx;
        sm.ml[WARPS][tid][1] = l;
        if (c.weight && tid < n_g) p.part[((size_t)t * p.heads + head0 + tid) * p.blocks + nb] = mx + log2f(l);
      }
      __syncthreads();
      for (int d = tid; d < HD; d += THREADS) {
        float acc[GH] = {};
        for (int i = max(0, j_min - base); i <= pos - base; ++i) {
          const float v = to_f32(sm.tail[1][i][d]);
#pragma unroll
          for (int k = 0; k < GH; ++k) acc[k] = fmaf(sm.tail_s[i][k], v, acc[k]);
        }
#pragma unroll
        for (int k = 0; k < GH; ++k) sm.tail_o[k][d] = acc[k];
      }
    }

    // ---- the finished blocks
    float o[DPL][2];
#pragma unroll
    for (int n = 0; n < DPL; ++n) o[n][0] = o[n][1] = 0.f;
    float ref = -INFINITY, l_row = 0.f;             // sums are relative to 2^ref; ref = running maximum - P_SHIFT
    for (int i = 0; i < n_mine; ++i) {
      if ((i & 31) == 0 && i > 0) {                 // the next 32 blocks; `at` holds the groups of even number, `at_next` the odd ones
        if ((i >> 5) & 1) look_up(i + 32, at, ks, vs); else look_up(i + 32, at_next, ks_next, vs_next);
      }
      issue(i + NSTAGE - 1);
      cp_wait<NSTAGE - 1>();
      __syncwarp();
      const bool odd = (i >> 5) & 1;
      const int a = __shfl_sync(0xffffffffu, odd ? at_next : at, i & 31);
      const float k_scale = __shfl_sync(0xffffffffu, odd ? ks_next : ks, i & 31), v_scale = __shfl_sync(0xffffffffu, odd ? vs_next : vs, i & 31);
      const int x = lo + warp + WARPS * i;
      if (a < 0) {                                   // a page that the pool does not have: the block counts for nothing
        if (c.weight && lane < n_g) p.part[((size_t)t * p.heads + head0 + lane) * p.blocks + x] = -INFINITY;
        continue;
      }
      const uint8_t *kt = sm.ring[warp][i % NSTAGE][0], *vt = sm.ring[warp][i % NSTAGE][1];
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int j = 0; j < HD / 64; ++j)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint4 w4 = *reinterpret_cast<const uint4*>(kt + k_chunk<HD>((n * 8 + g) * (HD / 16) + 4 * j + tq) * 16);
          const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t b0, b1;
            levels4<FMT>(w[e], b0, b1);
            mma_f16(sc[n], qf[4 * j + e], b0, b1);
          }
        }
      const float f = k_scale * row_scale;
      const int first = j_min - x * BLK;             // rows below are outside the window
      float v[2][2], mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          v[n][e] = n * 8 + tq * 2 + e >= first ? (sc[n][e] + sc[n][e + 2]) * f : -INFINITY;
          mx = fmaxf(mx, v[n][e]);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float ref_new = fmaxf(ref, mx - P_SHIFT);
      if (__any_sync(0xffffffffu, ref_new != ref)) {
        const float alpha = ref_new == ref ? 1.f : exp2f(ref - ref_new);
        ref = ref_new;
        l_row *= alpha;
#pragma unroll
        for (int n = 0; n < DPL; ++n) { o[n][0] *= alpha; o[n][1] *= alpha; }
      }
      float sum = 0.f, pr[2][2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          pr[n][e] = ref == -INFINITY ? (v[n][e] == v[n][e] ? 0.f : v[n][e]) : exp2f(v[n][e] - ref);
          sum += pr[n][e];
        }
      l_row += sum;
      if (c.weight) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (tq == 0 && g < n_g) p.part[((size_t)t * p.heads + head0 + g) * p.blocks + x] = ref + log2f(sum);
      }
      uint32_t pf[4];
      split2(pr[0][0], pr[0][1], pf[0], pf[1]);
      split2(pr[1][0], pr[1][1], pf[2], pf[3]);
      // values of rows 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9, dimensions [DPL g, DPL (g + 1))
      uint32_t vw[4][DPL / 4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int vr = 2 * tq + (r & 1) + 8 * (r >> 1);
        if (HD == 128) {
          const uint4 w4 = *reinterpret_cast<const uint4*>(vt + v_chunk<HD>(vr * 8 + g) * 16);
          vw[r][0] = w4.x; vw[r][1] = w4.y; vw[r][DPL / 4 - 2] = w4.z; vw[r][DPL / 4 - 1] = w4.w;
        } else {
          const uint2 w2 = *reinterpret_cast<const uint2*>(vt + v_chunk<HD>(vr * 4 + (g >> 1)) * 16 + (g & 1) * 8);
          vw[r][0] = w2.x; vw[r][1] = w2.y;
        }
      }
#pragma unroll
      for (int w = 0; w < DPL / 4; ++w)
#pragma unroll
        for (int y = 0; y < 2; ++y) {                // two dimensions at a time: bytes of two rows side by side
          const uint32_t sel = y ? 0x7362 : 0x5140;
          uint32_t b00, b01, b10, b11;
          levels4<FMT>(__byte_perm(vw[0][w], vw[1][w], sel), b00, b01);
          levels4<FMT>(__byte_perm(vw[2][w], vw[3][w], sel), b10, b11);
          float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16(c0, pf, b00, b10);
          mma_f16(c1, pf, b01, b11);
          const int n = 4 * w + 2 * y;
          o[n][0] = fmaf(v_scale, c0[0] + c0[2], o[n][0]);
          o[n][1] = fmaf(v_scale, c0[1] + c0[3], o[n][1]);
          o[n + 1][0] = fmaf(v_scale, c1[0] + c1[2], o[n + 1][0]);
          o[n + 1][1] = fmaf(v_scale, c1[1] + c1[3], o[n + 1][1]);
        }
      __syncwarp();                                  // the stage may be filled again
    }
    cp_wait<0>();
    __syncwarp();
    l_row += __shfl_xor_sync(0xffffffffu, l_row, 1);
    l_row += __shfl_xor_sync(0xffffffffu, l_row, 2);
    float* mine = reinterpret_cast<float*>(&sm.ring[warp][0][0][0]);       // [GH][HD]
#pragma unroll
    for (int n = 0; n < DPL; ++n) {
      mine[g * HD + DPL * (2 * tq) + n] = o[n][0];
      mine[g * HD + DPL * (2 * tq + 1) + n] = o[n][1];
    }
    if (tq == 0) { sm.ml[warp][g][0] = ref; sm.ml[warp][g][1] = l_row; }
    __syncthreads();

    // ---- the CTA's partial result: warps in their order, then the unfinished block
    const int parts = WARPS + (owner ? 1 : 0);
    for (int i = tid; i < n_g * HD; i += THREADS) {
      const int h = i / HD, d = i % HD;
      float mm = -INFINITY, ll = 0.f, acc = 0.f;
      for (int w = 0; w < parts; ++w) mm = fmaxf(mm, sm.ml[w][h][0]);
#pragma unroll
      for (int w = 0; w < WARPS + 1; ++w) {
        if (w == WARPS && !owner) break;
        const float f = sm.ml[w][h][0] == -INFINITY && mm == -INFINITY ? 1.f : exp2f(sm.ml[w][h][0] - mm);
        ll += f * sm.ml[w][h][1];
        acc += f * (w < WARPS ? reinterpret_cast<const float*>(&sm.ring[w][0][0][0])[h * HD + d] : sm.tail_o[h][d]);
      }
      sm.o[h][d] = acc;
      if (d == 0) { sm.oml[h][0] = mm; sm.oml[h][1] = ll; }
    }
    if (S > 1) cluster.sync(); else __syncthreads();

    // ---- the cluster's: every CTA an equal share of the outputs
    if (tid < n_g) {
      float mm = -INFINITY, ll = 0.f;
      for (int r = 0; r < S; ++r) mm = fmaxf(mm, S > 1 ? *cluster.map_shared_rank(&sm.oml[tid][0], r) : sm.oml[tid][0]);
      for (int r = 0; r < S; ++r) {
        const float m = S > 1 ? *cluster.map_shared_rank(&sm.oml[tid][0], r) : sm.oml[tid][0];
        const float l = S > 1 ? *cluster.map_shared_rank(&sm.oml[tid][1], r) : sm.oml[tid][1];
        ll += (m == -INFINITY && mm == -INFINITY ? 1.f : exp2f(m - mm)) * l;
      }
      sm.lse[tid][0] = mm;
      sm.lse[tid][1] = ll == 0.f ? 0.f : 1.f / ll;
    }
    __syncthreads();
    for (int i = rank * THREADS + tid; i < n_g * HD; i += S * THREADS) {
      const int h = i / HD, d = i % HD;
      const float mm = sm.lse[h][0];
      float acc = 0.f;
      for (int r = 0; r < S; ++r) {
        const float m = S > 1 ? *cluster.map_shared_rank(&sm.oml[h][0], r) : sm.oml[h][0];
        const float y = S > 1 ? *cluster.map_shared_rank(&sm.o[h][d], r) : sm.o[h][d];
        acc += (m == -INFINITY && mm == -INFINITY ? 1.f : exp2f(m - mm)) * y;
      }
      out[(size_t)g0 * HD + i] = from_f32<T>(acc * sm.lse[h][1]);
    }
    if (c.weight) {
      // weight of block x: the sum over the group's heads, in their order, of 2^(part - maximum) / sum
      const int end = owner ? nb + 1 : hi, begin = owner && lo >= nb ? nb : lo;
      for (int x = begin + tid; x < end; x += THREADS) {
        const int page = block_page(c, slot, x / per_page, p.err);
        if (page < 0) continue;
        const size_t i = ((size_t)page * c.kv_heads + kvh) * per_page + x % per_page;
        float w = g0 > 0 ? p.weight_out[i] : x == nb && pos == base ? 0.f : c.weight[i];
        for (int h = 0; h < n_g; ++h) w += exp2f(p.part[((size_t)t * p.heads + head0 + h) * p.blocks + x] - sm.lse[h][0]) * sm.lse[h][1];
        p.weight_out[i] = w;
      }
    }
    if (S > 1) cluster.sync(); else __syncthreads();      // nobody reads this CTA's results any more
  }

  if (owner && pos - base == BLK - 1) {              // the block is full: from the next step on it is read in 8 bits
    const int page = block_page(c, slot, nb / per_page, p.err);
    if (page >= 0) {
      const size_t i = ((size_t)page * c.kv_heads + kvh) * per_page + nb % per_page;
      finish_block<FMT>(&sm.tail[0][0][0], (const T*)nullptr, 0, BLK, HD, (uint8_t*)c.k + i * BLK * HD, c.k_scale + i, sm.red);
      finish_block<FMT>(&sm.tail[1][0][0], (const T*)nullptr, 0, BLK, HD, (uint8_t*)c.v + i * BLK * HD, c.v_scale + i, sm.red);
    }
  }
}

template <int HD, int FMT, typename T>
int launch(const BlockTcParams& p, const IertBatchView& b, const IertBlockView& c, int splits, cudaStream_t stream) {
  auto kernel = block_attention_tc_kernel<HD, FMT, T>;
  const size_t smem = sizeof(Shared<HD, T>);
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return iert_check_launch("block_attention (attributes)");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, c.kv_heads, b.n_seqs);
  cfg.blockDim = dim3(THREADS);
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

// `splits` (1, 2, 4, 8, 16; 0: by the rule below): CTAs that share a sequence's kv head.
IERT_API int iert_block_attention_tc(const void* qkv, void* out, const IertBatchView* batch, const IertBlockView* view, int heads, float scale,
                                     float* part, float* weight_out, const float* inv_freq, int rotary_dim, int pairing, float rot_mul, int splits,
                                     int* err, cudaStream_t stream) {
  if (batch->n_tokens <= 0) return IERT_OK;
  const IertBlockView& c = *view;
  if ((c.head_dim != 64 && c.head_dim != 128) || c.kv_heads <= 0 || heads <= 0 || heads % c.kv_heads || batch->n_tokens != batch->n_seqs ||
      batch->n_seqs > 65535 || c.kv_heads > 65535 || c.page_tokens <= 0 || c.page_tokens % BLK || c.table_width <= 0 || c.ring_pages <= 0 ||
      c.ring_pages > c.table_width || c.n_pages <= 0 || c.n_slots <= 0 || c.window < 0 ||
      (c.weight && (c.window || !part || !weight_out)) || ((uintptr_t)c.k | (uintptr_t)c.v) % 16 ||
      (inv_freq && (rotary_dim < 0 || rotary_dim > c.head_dim || (rotary_dim & 1) || (pairing != IERT_PAIR_HALF && pairing != IERT_PAIR_INTERLEAVED))))
    return IERT_BAD_ARGUMENT;
  if (splits < 0 || splits > 16 || (splits & (splits - 1))) return IERT_BAD_ARGUMENT;
  if (splits == 0) {
    const long long base = (long long)c.kv_heads * batch->n_seqs;
    splits = 1;
    while (splits < 16 && base * splits * 2 <= 3LL * iert_sm_count_cached()) splits *= 2;
  }
  BlockTcParams p = {};
  p.qkv = qkv; p.out = out; p.part = part; p.weight_out = weight_out;
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
