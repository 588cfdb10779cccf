// Penalties for repeated tokens, biases and a mask on a step's logits, and the best token that is left, in one pass:
//   x = logits[r, i];  i seen in row r's history: x / rep if x > 0 else x * rep
//   i among the history's answer, c > 0 times: x - freq * c - pres       (products and differences rounded one by one, in this order)
//   x + bias[i];  -infinity where the mask has no bit for i
// A cluster of up to eight CTAs shares a row: each owns a part of the vocabulary, counts the history's tokens that fall into it in
// shared memory, applies the rules to its logits and keeps the best; the bests meet in the first CTA's
// shared memory, which appends the choice to the row's history.  One launch, and nothing but the logits crosses the memory.
// Its bound is the logits' way from and to memory: a thread has its 16 logits of the next window on their way while it does those of
// this one (the first cross while the history is counted), and a cluster is as large as lets all rows run at once.  64 rows of
// 131,072 under all the rules take 26 us in clusters of four (38 in clusters of eight, two waves of them):
// 16.5 with no rule at all (67 MB, 10 us at the copy's rate, and one launch), and 4.3, 1.8 and 1.3 for histories of 4,096, masks and biases.
#include <cooperative_groups.h>

#include <utility>

#include "common.cuh"

namespace cg = cooperative_groups;
using namespace iert;

namespace {

constexpr int THREADS = 512, MAX_CLUSTER = 8;
constexpr int PER_THREAD = 16;                // logits of a thread in a window
constexpr int WINDOW = THREADS * PER_THREAD;
constexpr int PAST = 8;                       // tokens of the history a thread asks for at once
constexpr int COUNTED = 4 * WINDOW;           // ids whose counts stand in shared memory at a time

struct RulesParams {
  const float* logits; long long ld;
  float* out; long long ld_out;               // null: the rules' results are not written
  int vocab;
  int* history; int width, hist_rows;         // [hist_rows][width]
  const int *lens, *prompt_lens;              // [hist_rows]
  const int* rows;                            // history row of each logits row (null: its own number)
  const float* penalties;                     // [hist_rows][3]: repetition, presence, frequency; null: none
  const float* bias; long long ld_bias;       // 0: one row for all
  const uint32_t* mask; long long ld_mask;    // words of 32 ids, bit i % 32 of word i / 32; ld 0: one row for all
  int* chosen;                                // null: no choice is made
  int* lens_out;                              // null: nothing is appended
  int chunk;
  int* err;
};

__device__ __forceinline__ bool better(float v, int i, float bv, int bi) { return v > bv || (v == bv && i < bi); }

// Count: 16-bit words serve histories of up to 32,767 tokens (64 KB for the COUNTED ids), 32-bit words longer ones.  The highest bit: seen at all.
// VEC: rows, biases and results in 16-byte runs.
template <typename Count, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) logit_rules_kernel(RulesParams p) {
  extern __shared__ uint32_t words[];
  constexpr int PER_WORD = 4 / sizeof(Count);
  constexpr uint32_t SEEN = 1u << (8 * sizeof(Count) - 1);
  const Count* counts = reinterpret_cast<const Count*>(words);
  __shared__ float vs[THREADS / 32];
  __shared__ int is[THREADS / 32];
  __shared__ float best_v[MAX_CLUSTER];
  __shared__ int best_i[MAX_CLUSTER];
  cg::cluster_group cluster = cg::this_cluster();
  cg::cluster_group::arrival_token started;
  if (p.chosen) started = cluster.barrier_arrive();
  pdl_launch_dependents();
  pdl_wait();
  const int size = gridDim.x, rank = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* row = p.logits + (long long)r * p.ld;
  float* out = p.out ? p.out + (long long)r * p.ld_out : nullptr;
  const float* bias = p.bias ? p.bias + (long long)r * p.ld_bias : nullptr;
  const uint32_t* mask = p.mask ? p.mask + (long long)r * p.ld_mask : nullptr;
  const int lo = min(p.vocab, rank * p.chunk), hi = min(p.vocab, lo + p.chunk);
  // the k-th number of a thread in the window that begins with w0 (VEC: four neighbours at a time)
  auto id_of = [&](int w0, int k) { return VEC ? w0 + 4 * (tid + (k >> 2) * THREADS) + (k & 3) : w0 + tid + k * THREADS; };
  float next[PER_THREAD];
  auto load = [&](int w0) {
    const int w1 = min(hi, w0 + WINDOW);
#pragma unroll
    for (int k = 0; k < PER_THREAD; k += VEC ? 4 : 1) {
      const int i = id_of(w0, k);
      if (i >= w1) continue;
      if (VEC) {
        const float4 f = *reinterpret_cast<const float4*>(row + i);
        next[k] = f.x; next[k + 1] = f.y; next[k + 2] = f.z; next[k + 3] = f.w;
      } else {
        next[k] = row[i];
      }
    }
  };
  int h = p.rows ? p.rows[r] : r;
  load(lo);
  if (mask)                                   // this CTA's words, asked for now, are near when their windows come
    for (int i = lo + tid * 1024; i < hi; i += THREADS * 1024) asm volatile("prefetch.global.L2 [%0];" ::"l"(mask + (i >> 5)));
  if (h < 0 || h >= p.hist_rows) {            // no such history: the row is treated as one without
    if (p.hist_rows > 0 && rank == 0 && tid == 0) atomicOr(p.err, IERT_ERR_HISTORY);
    h = -1;
  }
  const bool counted = p.penalties && h >= 0;
  const int* hist = p.history + (long long)max(h, 0) * p.width;
  int past[PAST];                             // the first tokens, asked for together with the history's length
#pragma unroll
  for (int e = 0; e < PAST; ++e) past[e] = counted && tid + e * THREADS < p.width ? hist[tid + e * THREADS] : 0;
  const int len = h >= 0 ? min(max(p.lens[h], 0), p.width) : 0;
  const int prompt = h >= 0 ? p.prompt_lens[h] : 0;
  const float rep = counted ? p.penalties[3 * h] : 1.f, pres = counted ? p.penalties[3 * h + 1] : 0.f, freq = counted ? p.penalties[3 * h + 2] : 0.f;
  // Counts those of the history's tokens that are among the n ids from c0; the first PAST a thread come from registers for the first ids.
  auto count = [&](int c0, int n, bool first) {
    for (int i = tid; i < (n + 4 * PER_WORD - 1) / (4 * PER_WORD); i += THREADS) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto one = [&](int j, int token) {
      const int id = token - c0;
      if (id < 0 || id >= n) return;
      const int shift = PER_WORD == 1 ? 0 : 16 * (id % PER_WORD);
      if (j >= prompt) atomicAdd(&words[id / PER_WORD], 1u << shift); else atomicOr(&words[id / PER_WORD], SEEN << shift);
    };
    if (first) {
#pragma unroll
      for (int e = 0; e < PAST; ++e)
        if (tid + e * THREADS < len) one(tid + e * THREADS, past[e]);
    }
#pragma unroll 4
    for (int j = tid + (first ? PAST * THREADS : 0); j < len; j += THREADS) one(j, hist[j]);
    __syncthreads();
  };
  if (counted && lo < hi) count(lo, min(hi - lo, COUNTED), true);

  float bv = -INFINITY;
  int bi = 0x7fffffff;
  // A row's penalties are asked once, not each result: with these no NaN comes of them, and an infinity is the best of its thread.
  bool bad = counted && !(rep > 0.f && rep < INFINITY && fabsf(pres) < INFINITY && fabsf(freq) * (float)len < INFINITY);
  // Four logits at a time, most of which nothing happens to: what is common to the four is asked once (61 instructions a logit with each
  // rule asked of each, 64 rows of 131,072 then 32 us).  c: counts; m: a bit per allowed id; i, step: their ids.
  auto rules = [&](float (&y)[4], const uint32_t (&c)[4], const float (&b)[4], uint32_t m, int i, int step, int n) {
    uint32_t top = 0;                         // the model's logits are finite, as for the samplers; one that is ruled out may be anything
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, e < n && (m >> e & 1) ? __float_as_uint(y[e]) & 0x7fffffffu : 0u);
    bad |= top >= 0x7f800000u;
    if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!c[e]) continue;
        y[e] = y[e] > 0.f ? __fdiv_rn(y[e], rep) : __fmul_rn(y[e], rep);
        const uint32_t said = c[e] & ~SEEN;
        if (said) y[e] = __fsub_rn(__fsub_rn(y[e], __fmul_rn(freq, (float)said)), pres);
      }
    }
    if (bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = __fadd_rn(y[e], b[e]);         // -infinity rules an id out; +infinity or NaN is a mistake
        bad |= e < n && (m >> e & 1) && !(y[e] < INFINITY);
      }
    }
    if (m != 0xfu) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!(m >> e & 1)) y[e] = -INFINITY;
    }
    const float most = fmaxf(fmaxf(y[0], n > 1 ? y[1] : -INFINITY), fmaxf(n > 2 ? y[2] : -INFINITY, n > 3 ? y[3] : -INFINITY));
    if (most > bv) {                          // a thread meets its ids in their order: the first of equal ones stays
      bv = most;
      bi = i + (y[0] == most ? 0 : n > 1 && y[1] == most ? step : n > 2 && y[2] == most ? 2 * step : 3 * step);
    }
  };
  for (int w0 = lo; w0 < hi; w0 += WINDOW) {
    const int w1 = min(hi, w0 + WINDOW), c0 = lo + (w0 - lo) / COUNTED * COUNTED;      // the counts begin with id c0
    float x[PER_THREAD];
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k) x[k] = next[k];
    if (w1 < hi) load(w1);
    if (counted && w0 == c0 && w0 > lo) {
      __syncthreads();                        // the counts of the ids before are read
      count(c0, min(hi - c0, COUNTED), false);
    }
#pragma unroll
    for (int k = 0; k < PER_THREAD; k += 4) {
      const int i = id_of(w0, k);
      if (i >= w1) continue;
      uint32_t c[4] = {0, 0, 0, 0};
      float b[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {x[k], x[k + 1], x[k + 2], x[k + 3]};
      if (VEC) {
        if (counted) {
          if (PER_WORD == 2) {
            const uint2 q = *reinterpret_cast<const uint2*>(counts + (i - c0));
            c[0] = q.x & 0xffffu; c[1] = q.x >> 16; c[2] = q.y & 0xffffu; c[3] = q.y >> 16;
          } else {
            const uint4 q = *reinterpret_cast<const uint4*>(counts + (i - c0));
            c[0] = q.x; c[1] = q.y; c[2] = q.z; c[3] = q.w;
          }
        }
        if (bias) {
          const float4 f = __ldg(reinterpret_cast<const float4*>(bias + i));
          b[0] = f.x; b[1] = f.y; b[2] = f.z; b[3] = f.w;
        }
        rules(y, c, b, mask ? __ldg(mask + (i >> 5)) >> (i & 31) & 0xfu : 0xfu, i, 1, 4);
        if (out) *reinterpret_cast<float4*>(out + i) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
        const int n = min(4, (w1 - i + THREADS - 1) / THREADS);      // of the four that there are
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int id = i + e * THREADS;
          if (e >= n) continue;
          if (counted) c[e] = counts[id - c0];
          if (bias) b[e] = __ldg(bias + id);
          m |= (mask ? __ldg(mask + (id >> 5)) >> (id & 31) & 1u : 1u) << e;
        }
        rules(y, c, b, m, i, THREADS, n);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < n && out) out[i + e * THREADS] = y[e];
      }
    }
  }
  if (bad || bv == INFINITY) atomicOr(p.err, IERT_ERR_NONFINITE_LOGIT);
  if (!p.chosen) return;                      // (the same for the whole cluster)
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    if (better(ov, oi, bv, bi)) { bv = ov; bi = oi; }
  }
  if (lane == 0) { vs[warp] = bv; is[warp] = bi; }
  __syncthreads();
  cluster.barrier_wait(std::move(started));   // the first CTA runs: its shared memory may be written
  if (tid == 0) {
    for (int w = 1; w < THREADS / 32; ++w)
      if (better(vs[w], is[w], bv, bi)) { bv = vs[w]; bi = is[w]; }
    *cluster.map_shared_rank(&best_v[rank], 0) = bv;
    *cluster.map_shared_rank(&best_i[rank], 0) = bi;
  }
  cluster.sync();                             // every CTA has read the history's length by now
  if (rank != 0 || tid != 0) return;
  for (int c = 0; c < size; ++c)
    if (better(best_v[c], best_i[c], bv, bi)) { bv = best_v[c]; bi = best_i[c]; }
  if (bi == 0x7fffffff) {
    atomicOr(p.err, IERT_ERR_NOTHING_ALLOWED);
    bi = 0;
  }
  p.chosen[r] = bi;
  if (p.lens_out && h >= 0) {
    if (len < p.width) p.history[(long long)h * p.width + len] = bi;
    else atomicOr(p.err, IERT_ERR_HISTORY);
    p.lens_out[h] = min(len + 1, p.width);
  }
}

template <typename Count, bool VEC>
int launch(cudaLaunchConfig_t& cfg, const RulesParams& p) {
  if (cfg.dynamicSmemBytes > 40 * 1024 && !shared_memory_up_to<logit_rules_kernel<Count, VEC>>(COUNTED * sizeof(Count)))
    return iert_check_launch("logit_rules (shared memory)");
  cudaLaunchKernelEx(&cfg, logit_rules_kernel<Count, VEC>, p);
  return iert_check_launch("logit_rules");
}

__global__ void history_append_kernel(int* history, int width, int hist_rows, int* lens, const int* rows, const int* tokens, int n, int* err) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= n) return;
  const int h = rows ? rows[r] : r;
  if (h < 0 || h >= hist_rows || lens[h] < 0 || lens[h] >= width) {
    atomicOr(err, IERT_ERR_HISTORY);
    return;
  }
  history[(long long)h * width + lens[h]] = tokens[r];
  lens[h] += 1;
}

}  // namespace

IERT_API int iert_logit_rules(const float* logits, int rows_n, int vocab, long long ld, float* out, long long ld_out, int* history, int width,
                              int hist_rows, const int* lens, const int* prompt_lens, const int* rows, const float* penalties, const float* bias,
                              long long ld_bias, const void* mask, long long ld_mask, int* chosen, int* lens_out, int* err, cudaStream_t stream) {
  if (rows_n <= 0) return IERT_OK;
  if (vocab <= 0 || rows_n > 65535 || (hist_rows > 0 && (!history || !lens || !prompt_lens || width <= 0)) ||
      (hist_rows <= 0 && (penalties || lens_out)))
    return IERT_BAD_ARGUMENT;
  RulesParams p = {};
  p.logits = logits; p.ld = ld; p.out = out; p.ld_out = ld_out; p.vocab = vocab; p.history = history; p.width = width; p.hist_rows = hist_rows;
  p.lens = lens; p.prompt_lens = prompt_lens; p.rows = rows; p.penalties = penalties; p.bias = bias; p.ld_bias = ld_bias;
  p.mask = (const uint32_t*)mask; p.ld_mask = ld_mask; p.chosen = chosen; p.lens_out = lens_out; p.err = err;
  // as many CTAs a row, up to eight, as let all rows run at once (two CTAs an SM; clusters leave a tenth of the places empty)
  int cluster = MAX_CLUSTER;
  while (cluster > 1 && (long long)rows_n * cluster * 10 > 18LL * iert_sm_count_cached()) cluster >>= 1;
  // each CTA's share: whole runs of 128 ids (four words of the mask, 16-byte runs)
  const long long chunk = (((long long)vocab + cluster - 1) / cluster + 127) / 128 * 128;
  if (chunk * cluster > 0x7fffffffLL) return IERT_BAD_ARGUMENT;
  p.chunk = (int)chunk;
  const bool vec = vocab % 4 == 0 && ld % 4 == 0 && (uintptr_t)logits % 16 == 0 && (!out || (ld_out % 4 == 0 && (uintptr_t)out % 16 == 0)) &&
                   (!bias || (ld_bias % 4 == 0 && (uintptr_t)bias % 16 == 0));
  const bool small = width < 32768;
  const size_t smem = penalties ? (small ? 2 : 4) * (size_t)(p.chunk < COUNTED ? p.chunk : COUNTED) : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster, rows_n);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = iert_pdl_enabled ? 2 : 1;
  if (small) return vec ? launch<uint16_t, true>(cfg, p) : launch<uint16_t, false>(cfg, p);
  return vec ? launch<uint32_t, true>(cfg, p) : launch<uint32_t, false>(cfg, p);
}

// tokens[r] joins the history of row rows[r] (null: r); the rows are distinct.
IERT_API int iert_history_append(int* history, int width, int hist_rows, int* lens, const int* rows, const int* tokens, int n, int* err,
                                 cudaStream_t stream) {
  if (n <= 0) return IERT_OK;
  if (width <= 0 || hist_rows <= 0) return IERT_BAD_ARGUMENT;
  launch_dep(history_append_kernel, dim3((n + 127) / 128), dim3(128), 0, stream, history, width, hist_rows, lens, rows, tokens, n, err);
  return iert_check_launch("history_append");
}
