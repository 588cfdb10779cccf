// One-token attention over the 8-bit cache (block_cache.cuh) on the 5th-generation tensor cores: int8 levels, heads of 128, up to eight
// query heads to a key head.  (block_attention_tc.cu has the other forms.)
//
// tcgen05.mma multiplies 8-bit integers as they stand in shared memory, so no level is ever converted; the other operand is a
// number written in 8-bit digits, a column of the product per digit, and sums of 32-bit integers are exact:
//   S [128 positions x 32] = K [128 x 128] Q^T     Q: a head's query as fixed-point numbers, DIG signed digits of 7 bits (base 128)
//   O [128 dimensions x 32] += V^T [128 x 128] P   P: a head's probabilities times value scales as 32-bit fixed-point numbers, four unsigned digits of 8 bits
// A tile is eight blocks of 16 positions of a (sequence, kv head), keys row by row (K-major), the values' tile read with its columns as
// rows (MN-major).  Every position is one thread of the softmax, which needs about 265 instructions a warp and tile (mma.sync with
// its conversions: 3,400 for the same 128 positions): what remains is the stream of levels.
//   warps 0-3  softmax, a position per thread: a head's score from its digits, times the block's key scale; the probability times the
//              block's value scale, as digits, into (swizzled) shared memory.  A head's unit is a power of two of its own and goes by these
//              products alone, so that a block of large values that has no weight takes no digits from the others.  It moves where a tile's heaviest
//              product would pass 2^31 or lies below 2^P_LEAST; O is then read out, added up in registers and begun again.
//   then       two TMA producers, of keys and of values: page numbers (and scales) of 32 blocks at a time, one per lane; boxes of up to 128
//              positions, as a page's size allows, into a ring of tiles.
//   then       two MMA issuers, of the scores and of the weighted sums.  (One warp for both kinds of either took 1,450 cycles a tile: every
//              product, commit, copy and wait stands in one row there.)
// A cluster of up to 8 CTAs shares a (sequence, kv head): each takes a run of its blocks and adds up a share of the outputs from what
// the others have put into its shared memory.  Few long sequences need more CTAs than that to fill the device (an SM reads 42 GB/s at most, and
// clusters of 16 fit only seven of its eight groups of SMs): theirs are not clusters, put their results into scratch memory, and a
// second kernel, started while the first ends, adds them up (`WIDE`).  The unfinished block, up to 16 rows in the run's type, is done in fp32 by the
// last CTA, which also stores the step's own key and value and turns the block into levels when it is full.
// Queries as fixed-point numbers: bfloat16 runs 20 bits below the row's largest (three digits), float32 runs 27 (four).  A product of probability and value
// scale is off by at most half a unit, 2^-21 (bfloat16 runs; float32 runs 2^-25) of the heaviest one of its tile.
// Every wait is bounded; on expiry the kernel records IERT_ERR_WAIT_EXPIRED, waits (bounded) for its copies and MMAs, frees its TMEM
// and returns.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "block_cache.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace cg = cooperative_groups;
using namespace iert;
using namespace sm100;

namespace {

constexpr int HD = 128, TILE = 128, TILE_BLOCKS = TILE / BLK, GH = 8, SOFT = 128, MAX_SPLITS = 8, MERGE_THREADS = 128, MAX_PIECES = 160;
constexpr int TILE_BYTES = TILE * HD, BLOCK_BYTES = BLK * HD, NCOL = 32;
constexpr uint32_t TMEM_COLS = 128;            // S twice, O once per group
constexpr uint32_t WAIT_LIMIT = 1u << 22;
// Where a unit moves, the heaviest product of the tile goes to [2^(P_TOP - 1), 2^(P_TOP + 1)); 2^31 is the bound.  A tile whose heaviest lies below 2^P_LEAST
// moves it too.  Tiles may thus be lighter by 2^7, in float32 runs, which are to keep more bits, by 2^3, and heavier by 2^2.
constexpr int P_TOP = 28;
template <typename T> constexpr int P_LEAST = sizeof(T) == 4 ? 24 : 20;
constexpr float Y_TOP = 64.f;                  // a probability beyond moves its head's reference: its product with the largest scale there is still has a number
constexpr int MAX_RUN = 256;                   // tiles that O adds up at most: 255 * 127 * 128 * 256 < 2^31
constexpr int WIDE_FROM = 16384;               // positions that a sequence may hold from which few sequences' CTAs are no clusters
constexpr int TAIL_BLOCKS = 16;                // finished blocks that cost a CTA about as much time as the unfinished one

struct UmmaParams {
  const void* qkv;
  void* out;
  float* part;                 // [T][kv_heads][blocks][8]: base-2 logarithm of a block's unnormalised weight
  float* piece_o;              // WIDE: [T][kv_heads][CTAs][8][HD], what each CTA has
  float* piece_ml;             // and [T][kv_heads][CTAs][8][2], maximum and sum
  float* weight_out;
  int heads, blocks;
  int by_length;               // longest sequences first
  int run;                     // blocks of a box: they stand side by side in a page (1, 2, 4 or 8)
  float scale_log2e;
  const float* inv_freq;
  int rope, rotary_dim, pairing;
  float rot_mul;
  int* err;
};

template <typename T, int GROUPS, int NSTAGE> struct __align__(1024) Shared {
  // of the tiles' scales.  Those of tile i are written over when the keys of tile i + 4 have been used, which takes the scores of tile
  // i + 2 to have been read, by the group that read those of tile i before
  static constexpr int SLOTS = NSTAGE + 4;
  uint8_t ring[NSTAGE][2][TILE_BYTES];          // keys, values: rows of 128 bytes, 128-byte swizzle
  uint8_t qd[NCOL * HD];                         // digits of the queries: row 8 j + h is digit j of head h
  uint8_t pd[2][NCOL * TILE];                    // digits of the probabilities, likewise
  float q[GH][HD + 4];
  float o[GROUPS][GH][HD];                       // each group's finished blocks
  T tail[2][BLK][HD];
  float cs[HD];
  float tail_s[BLK][GH];
  float tail_o[GH][HD];
  float o_in[GH * HD + MAX_SPLITS];              // this CTA's share of the outputs, from every CTA of the cluster
  float ml_in[MAX_SPLITS][GH][2];
  float fac[MAX_SPLITS][GH];
  float ml[GROUPS + 1][GH][2];                   // maximum and sum: each group's blocks, the unfinished block
  float wfac[GROUPS + 1][GH];                    // what each of them counts for in the CTA's result
  float lse[GH][2];
  float rs[GH];                                  // what makes scores of the integers
  __align__(16) float top[GROUPS][2][4][GH];     // of each warp: largest scores, heaviest products
  __align__(16) uint32_t seen[GROUPS][2][4];     // of each warp, tiles in turn: see `softmax`
  float sum[GROUPS][4][GH];
  float2 scale[SLOTS][TILE_BLOCKS];              // key and value scale; a block that is not there, or in front of the window: key scale NaN of its own kind (see NOWHERE)
  uint32_t red[GROUPS * 4 + 4];
  uint64_t k_full[NSTAGE], v_full[NSTAGE], k_empty[NSTAGE], v_empty[NSTAGE], s_full[2], s_empty[2], p_ready[2], pv_done[2], drained;
  uint32_t tmem;
  int restart[2];
  int asked_k, asked_v;
  int abort_flag;
};
constexpr uint32_t NOWHERE = 0x7fc0beefu;        // the key scale of a block that counts for nothing (no division gives this pattern)

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 255u && *abort_flag) return false;
  }
  return false;
}
__device__ __forceinline__ void mma_i8(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
// A box of rows from `row` on, asked for by the lane of a converged warp whose `who` is set.
__device__ __forceinline__ void ask(uint32_t who, void* dst, const CUtensorMap* map, uint64_t* bar, int row) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
      ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(0), "r"(row), "r"(who) : "memory");
}
// s8 x (s8 or u8) -> s32, M x N; A MN-major on request, B K-major.
__host__ __device__ constexpr uint32_t instr_desc_i8(uint32_t M, uint32_t N, uint32_t b_signed, uint32_t a_mn) {
  return (2u << 4) | (1u << 7) | (b_signed << 10) | (a_mn << 15) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
// Barriers of one softmax group.
__device__ __forceinline__ void soft_sync(int group) { asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(SOFT) : "memory"); }
// All but the producer.
template <int N> __device__ __forceinline__ void early_sync() { asm volatile("bar.sync 3, %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  tmem_ld16_issue(taddr, r);
  tmem_ld16_issue(taddr + 16, r + 16);
  tmem_ld_wait();
}

// The largest of a number over the warp (NaN apart).
__device__ __forceinline__ float warp_top(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ float head_value(const T* src, int d, const UmmaParams& p, const float* cs) {
  const float x = to_f32(src[d]);
  if (!p.rope || d >= p.rotary_dim) return x;
  const int half = p.rotary_dim / 2;
  const bool second = p.pairing == IERT_PAIR_HALF ? d >= half : d & 1;
  const int k = p.pairing == IERT_PAIR_HALF ? (second ? d - half : d) : d >> 1;
  const float y = to_f32(src[p.pairing == IERT_PAIR_HALF ? (second ? d - half : d + half) : d ^ 1]);
  return to_f32(from_f32<T>(second ? y * cs[half + k] + x * cs[k] : x * cs[k] - y * cs[half + k]));
}

// GROUPS: of four softmax warps each, which take the tiles in turn and keep an O, references and sums of their own.  One group and two CTAs
// an SM where there are CTAs enough, else two groups and a deeper ring in one CTA an SM: a tile takes a group more than 1.1 us, an SM's share of the
// memory's rate brings one in 0.75 us.
template <typename T, int GROUPS, int NSTAGE, bool WIDE>
__global__ void __launch_bounds__(GROUPS * SOFT + 128, 3 - GROUPS)
block_attention_umma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, UmmaParams p, IertBatchView b,
                            IertBlockView c) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];        // no static shared memory: the window starts 1024-byte aligned
  using Sh = Shared<T, GROUPS, NSTAGE>;
  Sh& sm = *reinterpret_cast<Sh*>(smem_raw);
  constexpr int THREADS = GROUPS * SOFT + 128, KEYS = 4 * GROUPS, VALUES = KEYS + 1, SCORES = KEYS + 2, SUMS = KEYS + 3, SLOTS = Sh::SLOTS;
  static_assert(THREADS >= MAX_SPLITS * GH, "a thread per (CTA, head)");
  constexpr int DIG = sizeof(T) == 4 ? 4 : 3;
  cg::cluster_group cluster = cg::this_cluster();
  const int S = gridDim.x, rank = blockIdx.x;                  // the cluster is the grid's first axis
  const int kvh = blockIdx.y, n_g = p.heads / c.kv_heads;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int t = p.by_length ? rank_th_longest(b, blockIdx.z, reinterpret_cast<int*>(smem_raw)) : blockIdx.z;
  const int s = sequence_of_token(b, t);
  int slot = block_slot(c, b, s, p.err);
  if (slot >= 0 && !block_reaches(c, b.pos0[s], p.err)) slot = -1;
  T* out = (T*)p.out + ((size_t)t * p.heads + (size_t)kvh * n_g) * HD;
  if (slot < 0) {                                              // (the same for the whole cluster)
    pdl_launch_dependents();
    pdl_wait();
    if (rank == 0 && !WIDE)
      for (int i = tid; i < n_g * HD; i += THREADS) out[i] = from_f32<T>(0.f);
    return;
  }
  if (smem_addr(smem_raw) & 1023u) {                           // never expected; refuse rather than compute garbage
    if (tid == 0) atomicOr(p.err, IERT_ERR_WAIT_EXPIRED);
    return;
  }
  cg::cluster_group::arrival_token started;
  if (!WIDE) started = cluster.barrier_arrive();
  const int pos = b.pos0[s], nb = pos / BLK, base = nb * BLK, per_page = c.page_tokens / BLK;
  const int j_min = iert_first_visible(pos, c.window, 0), b_lo = min(j_min / BLK, nb) / p.run * p.run;
  // a run of blocks that begins with a box's first (blocks in front of the window's, or behind the last, count for nothing)
  const int per = ((nb - b_lo + (S > 1 ? TAIL_BLOCKS : 0) + S - 1) / S + p.run - 1) / p.run * p.run;
  const int lo = min(nb, b_lo + rank * per), hi = min(nb, lo + per);
  const int n_tiles = (hi - lo + TILE_BLOCKS - 1) / TILE_BLOCKS;
  const bool owner = rank == S - 1;                            // of the unfinished block
  const T* row = (const T*)p.qkv + (size_t)t * (size_t)(p.heads + 2 * c.kv_heads) * HD;
  volatile int* abort_flag = &sm.abort_flag;
  if (tid == 0) {
    for (int i = 0; i < NSTAGE; ++i) { mbar_init(&sm.k_full[i], 1); mbar_init(&sm.v_full[i], 1); mbar_init(&sm.k_empty[i], 1); mbar_init(&sm.v_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&sm.s_full[i], 1); mbar_init(&sm.s_empty[i], SOFT); mbar_init(&sm.p_ready[i], SOFT); mbar_init(&sm.pv_done[i], 1); }
    mbar_init(&sm.drained, 2);
    sm.abort_flag = 0; sm.asked_k = 0; sm.asked_v = 0;
    mbar_fence_init();
  }
  if (warp == SUMS) tmem_alloc(&sm.tmem, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();                                     // (a later kernel must not take the TMEM this CTA waits for)
  const uint32_t tmem = sm.tmem, o_col = 2 * NCOL;
  bool ok = true;

  // ---------------- TMA producers ----------------
  auto produce = [&](auto values) {
    constexpr bool V = decltype(values)::value;
    const CUtensorMap* map = V ? &map_v : &map_k;
    uint64_t *full = V ? sm.v_full : sm.k_full, *empty = V ? sm.v_empty : sm.k_empty;
    if (lane == 0) tma_prefetch_desc(map);
    const uint32_t leader = elect_leader();
    const int run = p.run, n_box = TILE_BLOCKS / run;
    // Pages of the 32 blocks after the next and scales of the next 32 are on their way while these 32 are asked for.  Like the step's
    // description, the page table does not depend on the kernel before.
    auto page_at = [&](int x) { return x < hi ? block_page(c, slot, x / per_page, p.err) : -1; };
    int at_next;
    float ks_next, vs_next;
    auto scales_at = [&](int x, int page) {
      at_next = page >= 0 ? (page * c.kv_heads + kvh) * per_page + x % per_page : -1;
      if (V) return;
      ks_next = __uint_as_float(NOWHERE); vs_next = 0.f;
      if (page >= 0 && x * BLK + BLK > j_min) {                // (a box may begin with blocks in front of the window: their levels are
        ks_next = c.k_scale[at_next];                          // fetched, and may be written meanwhile where a ring's newest block takes their
        vs_next = c.v_scale[at_next];                          // place, but count for nothing, whatever they are)
      }
    };
    const int page0 = page_at(lo + lane);
    int page = page_at(lo + 32 + lane);
    pdl_wait();
    scales_at(lo + lane, page0);
    int st = 0, slot_i = 0;
    uint32_t phase = 1;                                        // the stage's use before: there was none in the first round
    uint8_t* dst = sm.ring[0][V];
    for (int i0 = 0; i0 < n_tiles && ok; i0 += 32 / TILE_BLOCKS) {
      const int x = lo + i0 * TILE_BLOCKS + lane;
      const int at = at_next;
      const float2 scales = make_float2(ks_next, vs_next);
      scales_at(x + 32, page);
      page = page_at(x + 64);
      const unsigned heads_of_boxes = __ballot_sync(0xffffffffu, at >= 0 && (lane & (run - 1)) == 0);
#pragma unroll 1
      for (int k = 0; k < 32 / TILE_BLOCKS && i0 + k < n_tiles; ++k) {
        const int i = i0 + k;
        if (i >= NSTAGE && !__all_sync(0xffffffffu, wait_bar(&empty[st], phase, abort_flag))) { ok = false; break; }
        if (!V && (lane >> 3) == k) sm.scale[slot_i][lane & 7] = scales;
        if (!V) __syncwarp();
        if (lane == 0) {
          mbar_expect_tx(&full[st], __popc(heads_of_boxes >> (k * TILE_BLOCKS) & 0xffu) * run * BLOCK_BYTES);
          if (V) sm.asked_v = i + 1; else sm.asked_k = i + 1;
        }
        __syncwarp();
        for (int j = 0; j < n_box; ++j) {
          const int a = __shfl_sync(0xffffffffu, at, k * TILE_BLOCKS + j * run);
          ask(leader && a >= 0, dst + j * run * BLOCK_BYTES, map, &full[st], a * BLK);
        }
        if (++slot_i == SLOTS) slot_i = 0;
        dst += 2 * TILE_BYTES;
        if (++st == NSTAGE) { st = 0; phase ^= 1u; dst = sm.ring[0][V]; }
      }
    }
  };
  if (warp == KEYS) {
    produce(std::false_type());
  } else if (warp == VALUES) {
    produce(std::true_type());
  } else {
    // ---------------- the queries' digits (all warps but the producers) ----------------
    pdl_wait();
    const int me = warp > VALUES ? tid - 64 : tid;
    constexpr int N = GROUPS * SOFT + 64;
    if (p.rope) {
      const float where = (float)(pos + (c.shift ? c.shift[slot] : 0));
      for (int k = me; k < p.rotary_dim / 2; k += N) {
        float sn, co;
        sincosf(where * p.inv_freq[k], &sn, &co);
        sm.cs[k] = co * p.rot_mul;
        sm.cs[p.rotary_dim / 2 + k] = sn * p.rot_mul;
      }
      early_sync<N>();
    }
    if (owner) {
      const size_t off = ((size_t)slot * c.kv_heads + kvh) * BLK * HD;
      T *tk = (T*)c.tail_k + off, *tv = (T*)c.tail_v + off;
      const int old = (pos - base) * HD;
      constexpr int V = 16 / sizeof(T);
#pragma unroll 2
      for (int i = me * V; i < old; i += N * V) {
        const uint4 x = *reinterpret_cast<const uint4*>(tk + i), y = *reinterpret_cast<const uint4*>(tv + i);
        *reinterpret_cast<uint4*>(&sm.tail[0][0][0] + i) = x;
        *reinterpret_cast<uint4*>(&sm.tail[1][0][0] + i) = y;
      }
      const T *kn = row + (size_t)(p.heads + kvh) * HD, *vn = row + (size_t)(p.heads + c.kv_heads + kvh) * HD;
      for (int d = me; d < HD; d += N) {
        const T x = from_f32<T>(head_value(kn, d, p, sm.cs)), v = vn[d];
        sm.tail[0][pos - base][d] = x;
        sm.tail[1][pos - base][d] = v;
        tk[old + d] = x;
        tv[old + d] = v;
      }
    }
#pragma unroll 4
    for (int i = me; i < GH * HD; i += N) {
      const int r = i / HD, d = i % HD;
      sm.q[r][d] = r < n_g ? head_value(row + (size_t)r * HD + (size_t)kvh * n_g * HD, d, p, sm.cs) : 0.f;
    }
    early_sync<N>();
    for (int h = warp > VALUES ? warp - 2 : warp; h < GH; h += KEYS + 2) {       // a warp per head: four numbers a lane
      const float4 x = *reinterpret_cast<const float4*>(&sm.q[h][4 * lane]);
      uint32_t largest = max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w)));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
      // scaled by a power of two: the row's largest number lies in [2^TOP, 2^(TOP + 1))
      constexpr int TOP = DIG == 4 ? 26 : 19;
      const int e = min(max((int)(largest >> 23), TOP + 1), 253);
      const float f = __uint_as_float((uint32_t)(254 + TOP - e) << 23);
      // (what is not a number reaches the scores through the scale that turns integers into them)
      if (lane == 0) sm.rs[h] = (largest >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __uint_as_float((uint32_t)(e - TOP) << 23)) * p.scale_log2e;
      const int v[4] = {__float2int_rn(x.x * f), __float2int_rn(x.y * f), __float2int_rn(x.z * f), __float2int_rn(x.w * f)};
      uint32_t dig[4] = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        int y = v[k];
#pragma unroll
        for (int j = DIG - 1; j > 0; --j) {                    // the lowest digit stands last
          const int d = ((y + 64) & 127) - 64;
          dig[j] |= (uint32_t)(d & 255) << (8 * k);
          y = (y - d) >> 7;
        }
        dig[0] |= (uint32_t)(y & 255) << (8 * k);
      }
#pragma unroll
      for (int j = 0; j < DIG; ++j)
        *reinterpret_cast<uint32_t*>(sm.qd + (8 * j + h) * HD + (((lane >> 2) ^ (h & 7)) << 4) + (lane & 3) * 4) = dig[j];
    }
    fence_proxy_async_smem();
    early_sync<N>();

    if (warp >= SCORES) {
      // ---------------- MMA issuers (whole warps, one lane of each acting) ----------------
      constexpr uint32_t IDESC_S = instr_desc_i8(TILE, NCOL, 1, 0), IDESC_O = instr_desc_i8(HD, NCOL, 0, 1);
      const uint32_t leader = elect_leader();
      const uint32_t ring0 = smem_addr(sm.ring[0][0]);
      auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag)) != 0; };
      int st = 0;
      uint32_t phase = 0;                          // of stage st
      if (warp == SCORES) {
        const uint64_t qd = smem_desc_k128(smem_addr(sm.qd));
        for (int i = 0; i < n_tiles; ++i) {
          if (!warp_wait(&sm.k_full[st], phase) || (i >= 2 && !warp_wait(&sm.s_empty[i & 1], ((i >> 1) - 1) & 1))) { ok = false; break; }
          tc_fence_after();
          const uint64_t kd = smem_desc_k128(ring0 + st * 2 * TILE_BYTES);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_i8(leader, tmem + (i & 1) * NCOL, kd + k * 2, qd + k * 2, IDESC_S, k > 0);
          mma_commit(leader, &sm.s_full[i & 1]);
          mma_commit(leader, &sm.k_empty[st]);
          if (++st == NSTAGE) { st = 0; phase ^= 1u; }
        }
      } else {
        const uint64_t pd0 = smem_desc_k128(smem_addr(sm.pd[0]));
        for (int i = 0; i < n_tiles; ++i) {
          if (!warp_wait(&sm.v_full[st], phase) || !warp_wait(&sm.p_ready[i & 1], (i >> 1) & 1)) { ok = false; break; }
          tc_fence_after();
          const uint32_t more = *(volatile int*)&sm.restart[i & 1] ? 0u : 1u;
          const uint64_t vd = smem_desc_mn128(ring0 + (st * 2 + 1) * TILE_BYTES, TILE_BYTES), pd = pd0 + (i & 1) * (NCOL * TILE >> 4);
          const uint32_t o = tmem + o_col + (GROUPS == 2 ? (i & 1) * NCOL : 0);
          mma_i8(leader, o, vd, pd, IDESC_O, more);
#pragma unroll
          for (int k = 1; k < 4; ++k) mma_i8(leader, o, vd + k * (32 * HD >> 4), pd + k * 2, IDESC_O, 1u);
          mma_commit(leader, &sm.pv_done[i & 1]);
          mma_commit(leader, &sm.v_empty[st]);
          if (++st == NSTAGE) { st = 0; phase ^= 1u; }
        }
      }
      mma_commit(leader, &sm.drained);
    } else {
      // ---------------- the unfinished block, in fp32: a thread per (row, head), then per dimension ----------------
      const int grp = warp >> 2, me = tid & (SOFT - 1);            // position `me` of a tile; dimension `me` of O
      if (owner && grp == GROUPS - 1) {
        const int r = me >> 3, h = me & 7;
        float sc = -INFINITY;
        if (base + r <= pos && base + r >= j_min) {
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
        sm.tail_s[r][h] = sc;
        soft_sync(grp);
        float mx = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < BLK; ++i) mx = fmaxf(mx, sm.tail_s[i][h]);
        const float pr = mx == -INFINITY ? (sc == sc ? 0.f : sc) : ex2(sc - mx);
        soft_sync(grp);
        sm.tail_s[r][h] = pr;
        soft_sync(grp);
        if (r == 0) {
#pragma unroll
          for (int i = 0; i < BLK; ++i) l += sm.tail_s[i][h];
          sm.ml[GROUPS][h][0] = mx;
          sm.ml[GROUPS][h][1] = l;
          if (c.weight) p.part[(((size_t)t * c.kv_heads + kvh) * p.blocks + nb) * GH + h] = mx + log2f(l);
        }
        float acc[GH] = {};
        for (int i = max(0, j_min - base); i <= pos - base; ++i) {
          const float v = to_f32(sm.tail[1][i][me]);
#pragma unroll
          for (int k = 0; k < GH; ++k) acc[k] = fmaf(sm.tail_s[i][k], v, acc[k]);
        }
#pragma unroll
        for (int k = 0; k < GH; ++k) sm.tail_o[k][me] = acc[k];
      }

      // ---------------- softmax ----------------
      const uint32_t lane_bits = (uint32_t)((warp & 3) * 32) << 16, my_o = tmem + lane_bits + o_col + (GROUPS == 2 ? grp * NCOL : 0);
      const int blk = me >> 4;
      float* part = c.weight ? p.part + ((size_t)t * c.kv_heads + kvh) * p.blocks * GH : nullptr;
      // What a warp tells the others of a tile: a bit per head with a product of at least 2^P_LEAST, and whether a reference has to move, a product is too large
      // (or no number), a wait has run out.
      constexpr uint32_t HEADS = (1u << GH) - 1, MOVE = 1u << GH, LARGE = 2u << GH, GONE = 4u << GH;
      constexpr float LEAST = (float)(1u << P_LEAST<T>);
      float rs[GH], ref[GH], l[GH], acc[GH];
      float root[GH];                              // a product's unit is root^-2, a power of four: no factor on the way leaves fp32's range
#pragma unroll
      for (int h = 0; h < GH; ++h) { rs[h] = sm.rs[h]; ref[h] = -INFINITY; l[h] = 0.f; acc[h] = 0.f; root[h] = 1.f; }
      int run = 0;                                 // tiles in O
      // O of the tiles so far joins acc (dimension `me`)
      auto flush = [&](int i) {                    // i: the last tile in O
        if (!wait_bar(&sm.pv_done[i & 1], (i >> 1) & 1, abort_flag)) ok = false;
        __syncwarp();
        tc_fence_after();
        uint32_t r[32];
        tmem_ld32(my_o, r);
        tc_fence_before();
#pragma unroll
        for (int h = 0; h < GH; ++h) {
          const float hi2 = fmaf((float)(int)r[24 + h], 256.f, (float)(int)r[16 + h]), lo2 = fmaf((float)(int)r[8 + h], 256.f, (float)(int)r[h]);
          const float back = __uint_as_float((254u << 23) - __float_as_uint(root[h]));      // 1 / root
          acc[h] = fmaf(fmaf(hi2, 65536.f, lo2) * back, back, acc[h]);
        }
        run = 0;
      };
      for (int i = GROUPS == 2 ? grp : 0, turn = 0; i < n_tiles; i += GROUPS, turn ^= 1) {
        if (!wait_bar(&sm.s_full[i & 1], (i >> 1) & 1, abort_flag)) ok = false;
        __syncwarp();
        tc_fence_after();
        uint32_t r[32];
        tmem_ld32(tmem + lane_bits + (i & 1) * NCOL, r);
        const float2 sc = sm.scale[i % SLOTS][blk];
        tc_fence_before();
        mbar_arrive(&sm.s_empty[i & 1]);
        const int x = lo + i * TILE_BLOCKS + blk;
        const bool there = __float_as_uint(sc.x) != NOWHERE && x * BLK + (me & 15) >= j_min;
        const float v_scale = there ? sc.y : 0.f;
        float v[GH], y[GH], w[GH];
        uint32_t says = ok ? 0u : GONE;
#pragma unroll
        for (int h = 0; h < GH; ++h) {
          float f;
          if (DIG == 4) f = fmaf((float)((int)r[h] * 128 + (int)r[8 + h]), 16384.f, (float)((int)r[16 + h] * 128 + (int)r[24 + h]));
          else f = fmaf((float)((int)r[h] * 128 + (int)r[8 + h]), 128.f, (float)(int)r[16 + h]);
          v[h] = there ? f * (sc.x * rs[h]) : -INFINITY;
          y[h] = ex2(v[h] - ref[h]);
          w[h] = y[h] * v_scale * root[h] * root[h];
          if (!(y[h] <= Y_TOP)) says |= MOVE;
          if (!(w[h] < 2147483648.f)) says |= LARGE;
          if (w[h] >= LEAST) says |= 1u << h;
        }
        says = __reduce_or_sync(0xffffffffu, says);
        if (lane == 0) sm.seen[grp][turn][warp & 3] = says;
        soft_sync(grp);                            // (the other turn's words are written again only behind the next tile's barrier)
        const uint4 all = *reinterpret_cast<const uint4*>(&sm.seen[grp][turn][0]);
        says = all.x | all.y | all.z | all.w;
        if (says & GONE) { ok = false; break; }
        if ((says & (HEADS | MOVE | LARGE)) != HEADS || run == MAX_RUN) {        // (the same for all four warps)
          if (run > 0) flush(i - GROUPS);
          auto over_group = [&](const float (&z)[GH], int which) {               // the largest of the tile per head, for all to read
            float mx[GH];
#pragma unroll
            for (int h = 0; h < GH; ++h) mx[h] = warp_top(z[h]);
            if (lane == 0) {
              *reinterpret_cast<float4*>(&sm.top[grp][which][warp & 3][0]) = make_float4(mx[0], mx[1], mx[2], mx[3]);
              *reinterpret_cast<float4*>(&sm.top[grp][which][warp & 3][4]) = make_float4(mx[4], mx[5], mx[6], mx[7]);
            }
            soft_sync(grp);                        // (written again only behind another barrier of the group)
          };
          auto top = [&](int which, int h) {
            return fmaxf(fmaxf(sm.top[grp][which][0][h], sm.top[grp][which][1][h]), fmaxf(sm.top[grp][which][2][h], sm.top[grp][which][3][h]));
          };
          if (says & MOVE) {
            over_group(v, 0);
#pragma unroll
            for (int h = 0; h < GH; ++h) {
              const float to = fmaxf(ref[h], top(0, h));
              const float alpha = to == ref[h] ? 1.f : ex2(ref[h] - to);
              ref[h] = to;
              l[h] *= alpha;
              acc[h] *= alpha;
              y[h] = v[h] == -INFINITY ? 0.f : ex2(v[h] - to);
            }
          }
#pragma unroll
          for (int h = 0; h < GH; ++h) w[h] = y[h] * v_scale;
          over_group(w, 1);
#pragma unroll
          for (int h = 0; h < GH; ++h) {
            const int e = (int)(__float_as_uint(top(1, h)) >> 23);
            // 2^k with k even, the heaviest times which lies in [2^(P_TOP - 1), 2^(P_TOP + 1)); a tile without any leaves the unit as it is
            if (top(1, h) > 0.f) root[h] = __uint_as_float((uint32_t)(((P_TOP + 127 - max(e, 1)) >> 1) + 127) << 23);
            w[h] = w[h] * root[h] * root[h];
          }
        }
        if (i >= 2 && !wait_bar(&sm.pv_done[i & 1], ((i >> 1) - 1) & 1, abort_flag)) ok = false;      // the buffer is free
        uint8_t* pd = sm.pd[i & 1] + (me & 15);
#pragma unroll
        for (int h = 0; h < GH; ++h) {
          l[h] = fmaf(w[h], 0.f, l[h] + y[h]);     // (a value scale that is no number makes the head's sum none)
          const uint32_t z = __float2uint_rn(w[h]);
          uint8_t* at = pd + h * TILE + ((blk ^ h) << 4);
          at[0] = (uint8_t)z;
          at[8 * TILE] = (uint8_t)(z >> 8);
          at[16 * TILE] = (uint8_t)(z >> 16);
          at[24 * TILE] = (uint8_t)(z >> 24);
        }
        if (me == 0) sm.restart[i & 1] = run == 0;
        ++run;
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&sm.p_ready[i & 1]);
        if (part) {
          // sums over a block's 16 lanes, eight heads: halves of the heads are exchanged until a lane has one
          float a4[4], a2[2];
          const bool b8 = lane & 8, b4 = lane & 4, b2 = lane & 2;
#pragma unroll
          for (int h = 0; h < 4; ++h) a4[h] = (b8 ? y[4 + h] : y[h]) + __shfl_xor_sync(0xffffffffu, b8 ? y[h] : y[4 + h], 8);
#pragma unroll
          for (int h = 0; h < 2; ++h) a2[h] = (b4 ? a4[2 + h] : a4[h]) + __shfl_xor_sync(0xffffffffu, b4 ? a4[h] : a4[2 + h], 4);
          float one = (b2 ? a2[1] : a2[0]) + __shfl_xor_sync(0xffffffffu, b2 ? a2[0] : a2[1], 2);
          one += __shfl_xor_sync(0xffffffffu, one, 1);
          const float r4[4] = {b8 ? ref[4] : ref[0], b8 ? ref[5] : ref[1], b8 ? ref[6] : ref[2], b8 ? ref[7] : ref[3]};
          const float r2[2] = {b4 ? r4[2] : r4[0], b4 ? r4[3] : r4[1]};
          if (!(lane & 1) && x < hi) part[(size_t)x * GH + (b8 ? 4 : 0) + (b4 ? 2 : 0) + (b2 ? 1 : 0)] = (b2 ? r2[1] : r2[0]) + log2f(one);
        }
      }
      ok = __all_sync(0xffffffffu, ok) != 0;
      if (ok && run > 0) flush(GROUPS == 2 ? (n_tiles - 1 - grp) / 2 * 2 + grp : n_tiles - 1);       // its last tile
#pragma unroll
      for (int h = 0; h < GH; ++h) {
        sm.o[grp][h][me] = acc[h];
        float z = l[h];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        if (lane == 0) sm.sum[grp][warp & 3][h] = z;
      }
      if (me == 0)
#pragma unroll
        for (int h = 0; h < GH; ++h) sm.ml[grp][h][0] = ref[h];
    }
  }
  if (!ok && lane == 0) {
    atomicOr(p.err, IERT_ERR_WAIT_EXPIRED);
    *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && tid == 0) {                   // copies and MMAs still on their way end before the memory is let go
    mbar_wait(&sm.drained, 0, WAIT_LIMIT);
    for (int st = 0; st < NSTAGE; ++st) {
      if (sm.asked_k > st) mbar_wait(&sm.k_full[st], (((sm.asked_k - 1 - st) / NSTAGE)) & 1, WAIT_LIMIT);
      if (sm.asked_v > st) mbar_wait(&sm.v_full[st], (((sm.asked_v - 1 - st) / NSTAGE)) & 1, WAIT_LIMIT);
    }
  }
  if (tid < GH * GROUPS) {
    const int w = tid / GH, h = tid % GH;
    sm.ml[w][h][1] = (sm.sum[w][0][h] + sm.sum[w][1][h]) + (sm.sum[w][2][h] + sm.sum[w][3][h]);
  }
  __syncthreads();
  const int parts = GROUPS + (owner ? 1 : 0);
  if (tid < GH * (GROUPS + 1)) {
    const int w = tid / GH, h = tid % GH;
    float mm = -INFINITY;
    for (int k = 0; k < parts; ++k) mm = fmaxf(mm, sm.ml[k][h][0]);
    sm.wfac[w][h] = w >= parts ? 0.f : sm.ml[w][h][0] == mm ? 1.f : ex2(sm.ml[w][h][0] - mm);
  }
  if (!WIDE) cluster.barrier_wait(std::move(started));        // every CTA runs
  __syncthreads();
  if (warp == SUMS) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }

  if (WIDE) {
    const size_t piece = ((size_t)t * c.kv_heads + kvh) * S + rank;
    for (int i = tid; i < n_g * HD; i += THREADS) {
      const int h = i / HD, d = i % HD;
      float x = owner ? sm.wfac[GROUPS][h] * sm.tail_o[h][d] : 0.f;
#pragma unroll
      for (int w = 0; w < GROUPS; ++w) x += sm.wfac[w][h] * sm.o[w][h][d];
      p.piece_o[piece * GH * HD + i] = x;
    }
    if (tid < GH) {
      float mm = -INFINITY, ll = 0.f;
      for (int k = 0; k < parts; ++k) { mm = fmaxf(mm, sm.ml[k][tid][0]); ll += sm.wfac[k][tid] * sm.ml[k][tid][1]; }
      *reinterpret_cast<float2*>(p.piece_ml + (piece * GH + tid) * 2) = make_float2(mm, ll);
    }
  } else {
  // ---- the CTA's partial result, its groups' blocks and the unfinished one, goes to the CTAs that add up its pieces
  const int share = (n_g * HD + S - 1) / S;
  for (int i = tid; i < n_g * HD; i += THREADS) {
    const int h = i / HD, d = i % HD, to = i / share;
    float x = owner ? sm.wfac[GROUPS][h] * sm.tail_o[h][d] : 0.f;
#pragma unroll
    for (int w = 0; w < GROUPS; ++w) x += sm.wfac[w][h] * sm.o[w][h][d];
    cluster.map_shared_rank(&sm.o_in[0], to)[rank * share + i - to * share] = x;
  }
  if (tid < S * GH) {
    const int to = tid / GH, h = tid % GH;
    float mm = -INFINITY, ll = 0.f;
    for (int k = 0; k < parts; ++k) { mm = fmaxf(mm, sm.ml[k][h][0]); ll += sm.wfac[k][h] * sm.ml[k][h][1]; }
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
    float a = 0.f;
    for (int r = 0; r < S; ++r) a += sm.fac[r][i / HD] * sm.o_in[r * share + k];
    out[i] = from_f32<T>(a);
  }
  if (c.weight) {
    // weight of block x: the sum over the group's heads, in their order, of 2^(part - maximum) / sum
    const float* part = p.part + ((size_t)t * c.kv_heads + kvh) * p.blocks * GH;
    const int end = owner ? nb + 1 : hi;
    for (int x = lo + tid; x < end; x += THREADS) {
      const int page = block_page(c, slot, x / per_page, p.err);
      if (page < 0) continue;
      const size_t i = ((size_t)page * c.kv_heads + kvh) * per_page + x % per_page;
      float w = x == nb && pos == base ? 0.f : c.weight[i];
      const float4 a = *reinterpret_cast<const float4*>(part + (size_t)x * GH), b4 = *reinterpret_cast<const float4*>(part + (size_t)x * GH + 4);
      const float e[GH] = {a.x, a.y, a.z, a.w, b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int h = 0; h < GH; ++h)
        if (h < n_g) w += ex2(e[h] - sm.lse[h][0]) * sm.lse[h][1];
      p.weight_out[i] = w;
    }
  }
  }
  if (owner && pos - base == BLK - 1) {            // the block is full: from the next step on it is read in 8 bits
    const int page = block_page(c, slot, nb / per_page, p.err);
    if (page >= 0) {
      const size_t i = ((size_t)page * c.kv_heads + kvh) * per_page + nb % per_page;
      finish_block<IERT_LEVEL_INT8>(&sm.tail[0][0][0], HD, (uint8_t*)c.k + i * BLK * HD, c.k_scale + i, sm.red);
      finish_block<IERT_LEVEL_INT8>(&sm.tail[1][0][0], HD, (uint8_t*)c.v + i * BLK * HD, c.v_scale + i, sm.red);
    }
  }
}

// Adds up what the CTAs of a (sequence, kv head) have left, in their order, and the weights of its blocks.  The third axis of the grid
// shares a pair: columns of the outputs, and blocks.
template <typename T>
__global__ void __launch_bounds__(MERGE_THREADS) block_attention_umma_merge_kernel(UmmaParams p, IertBatchView b, IertBlockView c, int C) {
  __shared__ float fac[MAX_PIECES][GH];
  __shared__ float lse[GH][2];
  pdl_launch_dependents();
  const int kvh = blockIdx.x, s = blockIdx.y, z = blockIdx.z, Z = gridDim.z, tid = threadIdx.x;
  const int n_g = p.heads / c.kv_heads, per_page = c.page_tokens / BLK;
  int slot = block_slot(c, b, s, p.err);
  const int pos = b.pos0[s];
  if (slot >= 0 && !block_reaches(c, pos, p.err)) slot = -1;
  T* out = (T*)p.out + ((size_t)s * p.heads + (size_t)kvh * n_g) * HD;
  pdl_wait();
  if (slot < 0) {
    for (int i = z * MERGE_THREADS + tid; i < n_g * HD; i += Z * MERGE_THREADS) out[i] = from_f32<T>(0.f);
    return;
  }
  const float* ml = p.piece_ml + ((size_t)s * c.kv_heads + kvh) * C * GH * 2;
  const float* po = p.piece_o + ((size_t)s * c.kv_heads + kvh) * C * GH * HD;
  {                                                // sixteen threads per head
    const int h = tid >> 4, l16 = tid & 15;
    float mm = -INFINITY, ll = 0.f;
    for (int k = l16; k < C; k += 16) mm = fmaxf(mm, ml[(k * GH + h) * 2]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    for (int k = l16; k < C; k += 16) {
      const float2 x = *reinterpret_cast<const float2*>(ml + (k * GH + h) * 2);
      const float f = x.x == mm ? 1.f : ex2(x.x - mm);
      fac[k][h] = f;
      ll += f * x.y;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
    if (l16 == 0) { lse[h][0] = mm; lse[h][1] = ll == 0.f ? 0.f : 1.f / ll; }
  }
  __syncthreads();
  for (int i = z * MERGE_THREADS + tid; i < n_g * HD; i += Z * MERGE_THREADS) {
    float acc = 0.f;
#pragma unroll 8
    for (int k = 0; k < C; ++k) acc += fac[k][i / HD] * po[(size_t)k * GH * HD + i];
    out[i] = from_f32<T>(acc * lse[i / HD][1]);
  }
  if (c.weight) {
    const int nb = pos / BLK;
    const float* part = p.part + ((size_t)s * c.kv_heads + kvh) * p.blocks * GH;
    for (int x = z * MERGE_THREADS + tid; x <= nb; x += Z * MERGE_THREADS) {
      const int page = block_page(c, slot, x / per_page, p.err);
      if (page < 0) continue;
      const size_t i = ((size_t)page * c.kv_heads + kvh) * per_page + x % per_page;
      float w = x == nb && pos % BLK == 0 ? 0.f : c.weight[i];
      const float4 a = *reinterpret_cast<const float4*>(part + (size_t)x * GH), b4 = *reinterpret_cast<const float4*>(part + (size_t)x * GH + 4);
      const float e[GH] = {a.x, a.y, a.z, a.w, b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int h = 0; h < GH; ++h)
        if (h < n_g) w += ex2(e[h] - lse[h][0]) * lse[h][1];
      p.weight_out[i] = w;
    }
  }
}

// The levels of a pool as rows of 128 bytes, fetched as boxes of `run` blocks.
bool level_map(const void* levels, long long rows, int run, CUtensorMap* out) {
  tma_host::EncodeTiledFn fn = tma_host::encode_fn();
  if (!fn || rows <= 0 || rows > 0x7fffffffLL) return false;
  cuuint64_t dims[2] = {HD, (cuuint64_t)rows}, strides[1] = {HD};
  cuuint32_t box[2] = {HD, (cuuint32_t)(BLK * run)}, estr[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(levels), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Clusters of `size` CTAs that run at once: one CTA an SM, two softmax groups in it (GROUPS 2), or two with one.  Shared memory decides, and an empty
// kernel with as much is asked about: of one that takes tensor memory the runtime says one CTA an SM, though two run.
__global__ void room_kernel() {}
template <typename T, int GROUPS, int NSTAGE> int at_once(int size) {
  static int known[5];
  const size_t smem = sizeof(Shared<T, GROUPS, NSTAGE>);
  if (!known[0] && cudaFuncSetAttribute(room_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared<float, 2, 5>)) != cudaSuccess) return 1;
  return clusters_at_once(room_kernel, size, GROUPS * SOFT + 128, smem, known);
}

template <typename T, int GROUPS, int NSTAGE, bool WIDE>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const UmmaParams& p, const IertBatchView& b, const IertBlockView& c, int splits, cudaStream_t stream) {
  auto kernel = block_attention_umma_kernel<T, GROUPS, NSTAGE, WIDE>;
  const size_t smem = sizeof(Shared<T, GROUPS, NSTAGE>);
  static bool configured = false;
  if (!configured) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return iert_check_launch("block_attention (shared memory)");
    configured = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, c.kv_heads, b.n_seqs);
  cfg.blockDim = dim3(GROUPS * SOFT + 128);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (!WIDE) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = splits; attr[n].val.clusterDim.y = 1; attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (iert_pdl_enabled) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cudaLaunchKernelEx(&cfg, kernel, mk, mv, p, b, c);
  const int status = iert_check_launch("block_attention");
  if (status || !WIDE) return status;
  // a thread per output, and per block where weights are kept: a chain of three loads each (8 CTAs a pair took 10 us for 8,192 blocks)
  const int Z = c.weight ? std::min(64, std::max(8, p.blocks / MERGE_THREADS)) : 8;
  launch_dep(block_attention_umma_merge_kernel<T>, dim3(c.kv_heads, b.n_seqs, Z), dim3(MERGE_THREADS), 0, stream, p, b, c, splits);
  return iert_check_launch("block_attention (merge)");
}

template <typename T>
int launch(UmmaParams p, const IertBatchView& b, const IertBlockView& c, int splits, int groups, cudaStream_t stream) {
  const long long pairs = (long long)c.kv_heads * b.n_seqs, reach = (long long)c.ring_pages * c.page_tokens;         // the most that a sequence holds
  const int sms = iert_sm_count_cached();
  if (splits == 0) {
    // The largest clusters, up to eight, that all run at once with a CTA an SM (8 sequences of 2,048 positions with 8 key heads: 15.4, 12.9, 20.8 us
    // with 1, 2, 4 CTAs to a pair; two of 3,500: 17.3 us in clusters of eight, of which the device holds 15, and 10.8 of four).  Pairs that leave more
    // than eight SMs each, and may be long, take them all without a cluster (one sequence of 8,192 positions: 11.8 us, 10.6 as a cluster; 16,384: 14.3
    // and 15.1; 32,768: 20.1 and 23.6; 131,071: 53 and 78; two of 32,768: 26.0 and 26.4).
    if (pairs * (MAX_SPLITS + 1) <= sms && reach >= WIDE_FROM) splits = (int)(std::min(sms, MAX_PIECES) / pairs);
    else
      for (splits = MAX_SPLITS; splits > 1 && pairs > at_once<T, 2, 5>(splits);) splits >>= 1;
    // Twice the CTAs, two an SM with one group each, where they all run at once and sequences may be long enough for a second start (16 of 8,192, 128
    // pairs: 42.8 us, 38.5 so, of 4,096: 25.8 and 25.6, of 1,024: 13.5 and 14.4; 56 pairs of 14,000: 36.8 and 32.9, of 8,192: 24.1 and 22.9, of 3,500: 14.6 and
    // 15.5; 24 pairs of 30,000: 37.8 and 33.4, of 14,000: 21.8 and 22.0, of 7,000: 13.7 and 15.2; inside a model a start costs more: four layers, 8 sequences of 2,048 of at most 4,096: 448 us a step, 460 so).
    if (splits < MAX_SPLITS && groups != 2 && reach >= 4096 * splits && pairs <= at_once<T, 1, 2>(2 * splits)) splits *= 2;
  }
  const bool wide = splits > MAX_SPLITS;
  // Two groups where a CTA has an SM to itself, one where two share it (64 sequences of 4,096 positions: 82 us and 74).  Between one and two pairs an SM,
  // long sequences one after the other even out what the SMs have to do (24 of 4,096: 34.5 us for 39.0; 36 of 4,096: 45.2 and 44.7, of 8,192: 66.9 and
  // 74.7; 20 of 2,048: 24.9 and 24.5).
  if (groups == 0) groups = wide || pairs <= at_once<T, 2, 5>(splits) || (splits == 1 && pairs <= 2LL * sms && pairs * 3000 <= reach * sms) ? 2 : 1;
  p.by_length = pairs * splits > (groups == 2 ? sms : 2 * sms);      // (64 sequences of up to 4,096 positions: 83 us as they stand, 74 so)
  CUtensorMap mk, mv;
  const long long rows = (long long)c.n_pages * c.kv_heads * c.page_tokens;
  if (!level_map(c.k, rows, p.run, &mk) || !level_map(c.v, rows, p.run, &mv)) return IERT_BAD_ARGUMENT;
  if (wide) return launch<T, 2, 5, true>(mk, mv, p, b, c, splits, stream);
  return groups == 2 ? launch<T, 2, 5, false>(mk, mv, p, b, c, splits, stream) : launch<T, 1, 2, false>(mk, mv, p, b, c, splits, stream);
}

}  // namespace

// Floats of scratch for what the CTAs of a step leave for one another, in front of the blocks' weights.
IERT_API long long iert_block_attention_scratch() { return (long long)MAX_PIECES * GH * (HD + 2); }

// `splits`: CTAs that share a sequence's kv head (1, 2, 4, 8: a cluster; more: not); `groups` (1, 2) of softmax warps in each; 0: by rules.
// IERT_BAD_ARGUMENT: not a case of this kernel.
int block_attention_umma(const void* qkv, void* out, const IertBatchView* batch, const IertBlockView* view, int heads, float scale,
                         float* scratch, float* weight_out, const float* inv_freq, int rotary_dim, int pairing, float rot_mul, int splits,
                         int groups, int* err, cudaStream_t stream) {
  const IertBlockView& c = *view;
  if (c.head_dim != HD || c.format != IERT_LEVEL_INT8 || c.kv_heads <= 0 || heads <= 0 || heads % c.kv_heads || heads / c.kv_heads > GH ||
      batch->n_tokens != batch->n_seqs || batch->n_seqs > 65535 || c.kv_heads > 65535 || c.page_tokens <= 0 || c.page_tokens % BLK || c.table_width <= 0 ||
      c.ring_pages <= 0 || c.ring_pages > c.table_width || c.n_pages <= 0 || c.n_slots <= 0 || c.window < 0 ||
      !scratch || (c.weight && (c.window || !weight_out)) ||
      ((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.tail_k | (uintptr_t)c.tail_v | (uintptr_t)scratch) % 16 ||
      (inv_freq && (rotary_dim < 0 || rotary_dim > HD || (rotary_dim & 1) || (pairing != IERT_PAIR_HALF && pairing != IERT_PAIR_INTERLEAVED))))
    return IERT_BAD_ARGUMENT;
  const long long pairs = (long long)c.kv_heads * batch->n_seqs;
  if (splits < 0 || groups < 0 || groups > 2 || (splits > MAX_SPLITS ? pairs * splits > MAX_PIECES : (splits & (splits - 1)) != 0)) return IERT_BAD_ARGUMENT;
  // Few and short sequences are left to block_attention_tc.cu: its start overlaps the kernel in front and its end the one behind, which this one's shared and
  // tensor memory do not allow (four layers of a model with 8 key heads: one sequence of 700 positions 408 us a step, 418 here; of 12,000 445 and 451;
  // two of 7,000 452 and 465, of 12,000 507 and 503; three of 2,048 425 and 433, four 465 and 437; alone this kernel is the faster one by up to 1 us).
  if (splits == 0 && groups == 0 && pairs <= 24 && pairs * c.ring_pages * c.page_tokens < 120000) return IERT_BAD_ARGUMENT;
  UmmaParams p = {};
  p.run = TILE_BLOCKS;
  while ((c.page_tokens / BLK) % p.run) p.run >>= 1;
  p.qkv = qkv; p.out = out; p.weight_out = weight_out;
  p.piece_o = scratch; p.piece_ml = scratch + (long long)MAX_PIECES * GH * HD; p.part = scratch + iert_block_attention_scratch();
  p.heads = heads; p.blocks = c.table_width * (c.page_tokens / BLK);
  p.scale_log2e = scale * 1.44269504088896340736f;
  p.inv_freq = inv_freq; p.rope = inv_freq != nullptr; p.rotary_dim = rotary_dim; p.pairing = pairing; p.rot_mul = rot_mul; p.err = err;
  return c.tail_dtype == IERT_BF16 ? launch<__nv_bfloat16>(p, *batch, c, splits, groups, stream) : launch<float>(p, *batch, c, splits, groups, stream);
}
