// Beam search on the device: the selection over beams x vocabulary
// (fcu_beam_step) and the reordering of the beams' caches after it
// (fcu_cache_reorder).  The reference samples one sequence on the host
// (src/L8/sampling.js:28-96) and has no beam search.
#include "common.cuh"

namespace fcu {
namespace {

// ------------------------------------------------------------------ selection
// Two kernels.  beam_rows reads every logit once: a CTA takes one slice of one
// row, keeps the slice's running maximum and sum of exponentials and its W
// best (logit, token) pairs.  beam_merge, one CTA per sequence, turns the
// slices' sums into each row's log-sum-exp and picks the W best of the
// W x slices x W survivors.  Within a row the order of the candidates is the
// order of the logits, so W per slice are enough.  The bound is reading the
// logits (HBM).
constexpr int kBeamThreads = 256;
constexpr int kMaxW = 32;
constexpr int kPer = 16;                            // logits a thread holds at a time
constexpr int kTile = kBeamThreads * kPer;
constexpr int kMaxSlices = 64;

using Key = unsigned long long;

// Larger logit, larger key; equal logits (0 and -0 too), lower token first.
// NaN is below -inf; 0 is below every key.
__device__ __forceinline__ Key beam_key(float x, uint32_t token) {
  uint32_t u = __float_as_uint(x + 0.0f);
  u = u & 0x80000000u ? ~u : u | 0x80000000u;
  if (x != x) u = 1;
  return (Key)u << 32 | (0xffffffffu - token);
}

struct BeamArgs {
  const float *logits;
  int64_t ld;
  const float *scores;
  const uint8_t *done;
  int64_t V;
  int B, W, eos, slices;
  int64_t slice;         // logits per slice
  float2 *sums;          // [rows][slices] maximum, sum of exp(x - maximum)
  Key *best;             // [rows][slices][W]
  float *out_scores;
  int32_t *tokens, *parents;
  uint8_t *out_done;
};

__global__ void __launch_bounds__(kBeamThreads) beam_rows_kernel(BeamArgs a) {
  pdl_trigger();
  __shared__ Key tops[kBeamThreads];
  __shared__ Key pool[kMaxW * (kPer + 1)];   // the W best so far, then a tile's newcomers
  __shared__ Key sorted[kMaxW];
  __shared__ int count;
  __shared__ float red_m[kBeamThreads / 32], red_s[kBeamThreads / 32];
  const int tid = threadIdx.x, W = a.W;
  const int64_t row = blockIdx.y;
  const int64_t v0 = (int64_t)blockIdx.x * a.slice, v1 = min(a.V, v0 + a.slice);
  if (tid < W) sorted[tid] = 0;
  pdl_wait();
  const float *x = a.logits + row * a.ld;
  float m = -INFINITY, s = 0.f;
  bool nan = false;
  Key bar = 0;                               // the W-th best so far
  __syncthreads();
  for (int64_t t0 = v0; t0 < v1; t0 += kTile) {
    float f[kPer];
    Key top = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int64_t v = t0 + i * kBeamThreads + tid;
      f[i] = v < v1 ? x[v] : -INFINITY;
    }
    float tm = m;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int64_t v = t0 + i * kBeamThreads + tid;
      nan |= f[i] != f[i];
      tm = fmaxf(tm, f[i]);
      if (v < v1) {
        const Key k = beam_key(f[i], (uint32_t)v);
        top = k > top ? k : top;
      }
    }
    if (tm > -INFINITY) {
      s *= expf(m - tm);
      float ts = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; i++) ts += expf(f[i] - tm);
      s += ts;
      m = tm;
    }
    if (!__syncthreads_or(top > bar)) continue;
    // Of the threads' best keys the W largest bound the tile's W best from
    // below, and only their threads can hold one of those.
    tops[tid] = top;
    if (tid == 0) count = W;
    if (tid < W) pool[tid] = sorted[tid];
    __syncthreads();
    if (top > bar) {
      int above = 0;
      for (int i = 0; i < kBeamThreads; i++) above += tops[i] > top;
      if (above < W)
#pragma unroll
        for (int i = 0; i < kPer; i++) {
          const int64_t v = t0 + i * kBeamThreads + tid;
          if (v < v1) {
            const Key k = beam_key(f[i], (uint32_t)v);
            if (k > bar) pool[atomicAdd(&count, 1)] = k;
          }
        }
    }
    __syncthreads();
    const int n = count;
    for (int i = tid; i < n; i += kBeamThreads) {
      const Key k = pool[i];
      int above = 0;
      for (int j = 0; j < n; j++) above += pool[j] > k;
      if (above < W && k) sorted[above] = k;
    }
    __syncthreads();
    bar = sorted[W - 1];
  }
  // the slice's maximum and sum: lanes, then warps, in a fixed order
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    const float M = fmaxf(m, om);
    s = M > -INFINITY ? s * expf(m - M) + os * expf(om - M) : 0.f;
    m = M;
  }
  nan = __syncthreads_or(nan);
  if ((tid & 31) == 0) red_m[tid >> 5] = m, red_s[tid >> 5] = s;
  __syncthreads();
  const int64_t at = row * a.slices + blockIdx.x;
  if (tid == 0) {
    float M = -INFINITY, S = 0.f;
    for (int w = 0; w < kBeamThreads / 32; w++) M = fmaxf(M, red_m[w]);
    for (int w = 0; w < kBeamThreads / 32; w++) S += M > -INFINITY ? red_s[w] * expf(red_m[w] - M) : 0.f;
    a.sums[at] = make_float2(M, nan ? NAN : S);
  }
  if (tid < W) a.best[at * W + tid] = sorted[tid];
}

// A candidate of the merge: score, then lowest w * V + token.
struct Cand {
  double score;
  int64_t flat;
};
__device__ __forceinline__ bool beats(const Cand &x, const Cand &y) {
  return x.score > y.score || (x.score == y.score && x.flat < y.flat);
}

__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(BeamArgs a) {
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t dyn[];
  Cand *cand = reinterpret_cast<Cand *>(dyn);          // [W * slices * W]
  __shared__ Cand tops[kBeamThreads];
  __shared__ double lse[kMaxW];
  __shared__ int picked[kBeamThreads], npicked;
  const int tid = threadIdx.x, W = a.W;
  const int64_t b = blockIdx.x;
  pdl_wait();
  if (tid == 0) npicked = 0;
  for (int w = tid; w < W; w += kBeamThreads) {
    const float2 *sm = a.sums + (b * W + w) * a.slices;
    float M = -INFINITY;
    for (int i = 0; i < a.slices; i++) M = fmaxf(M, sm[i].x);
    double S = 0;
    for (int i = 0; i < a.slices; i++) S += sm[i].x > -INFINITY || sm[i].y != sm[i].y ? sm[i].y * exp((double)sm[i].x - M) : 0.0;
    lse[w] = (double)M + log(S);
  }
  __syncthreads();
  const int per = a.slices * W, N = W * per;
  for (int i = tid; i < N; i += kBeamThreads) {
    const int w = i / per, r = i - w * per;
    const int64_t row = b * W + w;
    const double cum = a.scores[row];
    const bool done = a.done[row] != 0;
    // beams with nothing finite to offer stand for their lowest tokens
    const bool dead = !isfinite(cum) || (!done && !isfinite(lse[w]));
    Cand c{-INFINITY, INT64_MAX};
    if (done || dead) {
      // eos first, then the other tokens in order; only W of them can count
      int64_t token = r;
      if (done && !dead) token = r == 0 ? a.eos : r - (r <= a.eos);
      if (r < W && token < a.V) {
        c.score = done && !dead && r == 0 ? cum : -INFINITY;
        c.flat = (int64_t)w * a.V + token;
      }
    } else {
      const Key k = a.best[row * per + r];
      if (k) {
        const uint32_t token = 0xffffffffu - (uint32_t)k, u = (uint32_t)(k >> 32);
        const float x = __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);   // beam_key's logit back
        const double v = cum + ((double)x - lse[w]);
        c.score = isfinite(v) ? v : -INFINITY;
        c.flat = (int64_t)w * a.V + token;
      }
    }
    cand[i] = c;
  }
  __syncthreads();
  // the threads whose best is among the W best of those
  Cand top{-INFINITY, INT64_MAX};
  for (int i = tid; i < N; i += kBeamThreads)
    if (beats(cand[i], top)) top = cand[i];
  tops[tid] = top;
  __syncthreads();
  int above = 0;
  for (int i = 0; i < kBeamThreads; i++) above += beats(tops[i], top);
  if (above < W && top.flat != INT64_MAX) picked[atomicAdd(&npicked, 1)] = tid;
  __syncthreads();
  // every candidate of those threads against every other
  const int rounds = (N + kBeamThreads - 1) / kBeamThreads, np = npicked;
  for (int i = tid; i < np * rounds; i += kBeamThreads) {
    const int me = picked[i % np] + i / np * kBeamThreads;
    if (me >= N || cand[me].flat == INT64_MAX) continue;
    const Cand c = cand[me];
    int rank = 0;
    for (int p = 0; p < np && rank < W; p++)
      for (int q = picked[p]; q < N; q += kBeamThreads) rank += beats(cand[q], c);
    if (rank < W) {
      const int w = (int)(c.flat / a.V);
      const int64_t o = b * W + rank;
      const int32_t token = (int32_t)(c.flat - (int64_t)w * a.V);
      a.out_scores[o] = (float)c.score;
      a.tokens[o] = token;
      a.parents[o] = w;
      a.out_done[o] = a.done[b * W + w] != 0 || token == a.eos;
    }
  }
}

// Slices per row: enough CTAs for four per SM, of at least half a tile each.
int beam_slices(int num_sms, int64_t rows, int64_t V) {
  int64_t s = (4 * (int64_t)num_sms + rows - 1) / (rows > 0 ? rows : 1);
  const int64_t most = (V + kTile / 2 - 1) / (kTile / 2);
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : s > kMaxSlices ? kMaxSlices : s);
}

// The merge holds W * slices * W candidates in shared memory.
int beam_plan(int num_sms, int B, int W, int64_t V) {
  int s = beam_slices(num_sms, (int64_t)B * W, V);
  while (s > 1 && (size_t)W * W * s * sizeof(Cand) > 160 * 1024) s--;
  return s;
}

// ------------------------------------------------------------------ reordering
// A thread owns 16 bytes at one place of every beam of a sequence: it reads
// them from the beams that another beam continues, then writes the beams that
// continue another.  No other thread touches that place, so the permutation
// (with repetitions) is done in place without a wait.
constexpr int kReThreads = 128;

struct ReArgs {
  uint8_t *base[8];
  int64_t heads[8], unit[8];
  int n_arrays;
  int64_t layers, blocks;
  const int32_t *table, *parents, *lens;
  int bs, mb, B, W;
  int64_t cap;
};

__device__ __forceinline__ int64_t re_block(const ReArgs &a, int64_t r, int64_t i) {
  if (!a.table) return r * a.mb + i;
  const int64_t p = a.table[r * a.mb + i];
  return p >= 0 && p < a.blocks ? p : -1;
}

// copies [off, off + n) bytes of a block's head segment, n <= 16, off and n multiples of 4
__device__ __forceinline__ void re_load(uint4 *dst, const uint8_t *src, int n, bool wide) {
  if (wide && n == 16) {
    *dst = *reinterpret_cast<const uint4 *>(src);
  } else {
    uint32_t *d = reinterpret_cast<uint32_t *>(dst);
    for (int i = 0; 4 * i < n; i++) d[i] = reinterpret_cast<const uint32_t *>(src)[i];
  }
}
__device__ __forceinline__ void re_store(uint8_t *dst, const uint4 *src, int n, bool wide) {
  if (wide && n == 16) {
    *reinterpret_cast<uint4 *>(dst) = *src;
  } else {
    const uint32_t *s = reinterpret_cast<const uint32_t *>(src);
    for (int i = 0; 4 * i < n; i++) reinterpret_cast<uint32_t *>(dst)[i] = s[i];
  }
}

__global__ void __launch_bounds__(kReThreads) cache_reorder_kernel(ReArgs a) {
  pdl_trigger();
  extern __shared__ __align__(16) uint4 hold[];     // [W][kReThreads]
  __shared__ int src_s[kMaxW];                      // the beam each one becomes; itself if it stays
  __shared__ int64_t len_s[kMaxW];
  __shared__ uint32_t needed_s;
  const int tid = threadIdx.x, W = a.W;
  const int b = blockIdx.y;
  const int64_t layer = blockIdx.z;
  pdl_wait();
  if (tid < W) {
    const int p = a.parents[(int64_t)b * W + tid];
    src_s[tid] = p >= 0 && p < W ? p : tid;
    const int64_t n = a.lens[(int64_t)b * W + tid];
    len_s[tid] = n < 0 ? 0 : n > a.cap ? a.cap : n;
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t needed = 0;
    for (int w = 0; w < W; w++)
      if (src_s[w] != w) needed |= 1u << src_s[w];
    needed_s = needed;
  }
  __syncthreads();
  const uint32_t needed = needed_s;
  if (!needed) return;
  int64_t longest = 0;
  for (int w = 0; w < W; w++)
    if (needed >> w & 1) longest = max(longest, len_s[w]);
  for (int x = 0; x < a.n_arrays; x++) {
    const int64_t unit = a.unit[x], seg = a.bs * unit;      // bytes of one head of one block
    const bool wide = seg % 16 == 0;
    const int per_seg = (int)((seg + 15) / 16);             // pieces of one segment
    const int64_t segs = (longest + a.bs - 1) / a.bs;
    const int64_t pieces = a.heads[x] * segs * per_seg;
    for (int64_t i = (int64_t)blockIdx.x * kReThreads + tid; i < pieces; i += (int64_t)gridDim.x * kReThreads) {
      const int64_t hs = i / per_seg, off = (i - hs * per_seg) * 16;
      const int64_t h = hs / segs, blk = hs - h * segs;
      for (uint32_t m = needed; m; m &= m - 1) {
        const int w = __ffs(m) - 1;
        const int64_t p = re_block(a, (int64_t)b * W + w, blk);
        const int n = (int)min(min((int64_t)16, seg - off), (len_s[w] - blk * a.bs) * unit - off);
        if (p >= 0 && n > 0)
          re_load(hold + w * kReThreads + tid, a.base[x] + ((layer * a.blocks + p) * a.heads[x] + h) * seg + off, n, wide);
      }
      for (int w = 0; w < W; w++) {
        const int src = src_s[w];
        if (src == w) continue;
        const int64_t p = re_block(a, (int64_t)b * W + w, blk), ps = re_block(a, (int64_t)b * W + src, blk);
        const int n = (int)min(min((int64_t)16, seg - off), (len_s[src] - blk * a.bs) * unit - off);
        if (p >= 0 && ps >= 0 && n > 0)
          re_store(a.base[x] + ((layer * a.blocks + p) * a.heads[x] + h) * seg + off, hold + src * kReThreads + tid, n, wide);
      }
    }
  }
}

}  // namespace
}  // namespace fcu

using namespace fcu;

extern "C" {

int64_t fcu_beam_work(fcu_ctx *ctx, int B, int W, int64_t V) {
  if (!ctx || B < 0 || W < 1 || W > kMaxW || V < 1) return -1;
  const int64_t parts = (int64_t)B * W * beam_plan(ctx->num_sms, B, W, V);
  return parts * (sizeof(float2) + W * sizeof(Key));
}

int fcu_beam_step(fcu_ctx *ctx, const float *logits, int64_t ld, const float *scores, const uint8_t *done, int B,
                  int W, int64_t V, int eos, float *out_scores, int32_t *tokens, int32_t *parents,
                  uint8_t *out_done, void *work, int64_t work_bytes) {
  FCU_CTX(ctx);
  FCU_REQUIRE(B >= 0 && W >= 1 && W <= kMaxW, "fcu_beam_step: %d sequences of %d beams (1..%d)", B, W, kMaxW);
  FCU_REQUIRE(V >= 1 && V <= INT_MAX, "fcu_beam_step: a vocabulary of %lld", (long long)V);
  FCU_REQUIRE(eos >= 0 && eos < V, "fcu_beam_step: eos %d outside the vocabulary", eos);
  FCU_REQUIRE(ld >= V, "fcu_beam_step: row stride %lld too small", (long long)ld);
  FCU_REQUIRE((int64_t)B * W <= 65535, "fcu_beam_step: %d x %d rows in one call", B, W);
  if (B == 0) return FCU_OK;
  FCU_REQUIRE(logits && scores && done && out_scores && tokens && parents && out_done, "fcu_beam_step: null pointer");
  FCU_REQUIRE((const void *)out_scores != scores && out_done != done, "fcu_beam_step: an output is an input");
  const int64_t need = fcu_beam_work(ctx, B, W, V);
  FCU_REQUIRE(work && work_bytes >= need && ((uintptr_t)work & 15) == 0,
              "fcu_beam_step: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)need);
  BeamArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.scores = scores;
  a.done = done;
  a.V = V;
  a.B = B;
  a.W = W;
  a.eos = eos;
  a.slices = beam_plan(ctx->num_sms, B, W, V);
  a.slice = (V + a.slices - 1) / a.slices;
  a.best = (Key *)work;
  a.sums = (float2 *)(a.best + (int64_t)B * W * a.slices * W);
  a.out_scores = out_scores;
  a.tokens = tokens;
  a.parents = parents;
  a.out_done = out_done;
  const size_t smem = (size_t)W * W * a.slices * sizeof(Cand);
  static bool set[64] = {false};
  if (!set[ctx->device & 63]) {
    FCU_CHECK_CUDA(cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    set[ctx->device & 63] = true;
  }
  FCU_CHECK_CUDA(launch_pdl(beam_rows_kernel, dim3(a.slices, B * W), dim3(kBeamThreads), 0, ctx->stream, a));
  note_launch();
  FCU_CHECK_CUDA(launch_pdl(beam_merge_kernel, dim3(B), dim3(kBeamThreads), smem, ctx->stream, a));
  note_launch();
  return FCU_OK;
}

int fcu_cache_reorder(fcu_ctx *ctx, const fcu_cache_array *arrays, int n_arrays, int64_t layers, int64_t blocks,
                      const int32_t *table, int block_size, int max_blocks, const int32_t *parents,
                      const int32_t *lens, int B, int W) {
  FCU_CTX(ctx);
  FCU_REQUIRE(B >= 0 && B <= 65535 && W >= 1 && W <= kMaxW, "fcu_cache_reorder: %d sequences of %d beams (1..%d)", B, W,
              kMaxW);
  FCU_REQUIRE(n_arrays >= 0 && n_arrays <= 8 && (arrays || n_arrays == 0), "fcu_cache_reorder: %d arrays (at most 8)",
              n_arrays);
  FCU_REQUIRE(layers >= 0 && layers <= 65535 && blocks >= 0 && block_size > 0 && max_blocks > 0,
              "fcu_cache_reorder: bad cache geometry");
  FCU_REQUIRE(table || (int64_t)B * W * max_blocks <= blocks, "fcu_cache_reorder: %d beams of %d blocks in %lld blocks",
              B * W, max_blocks, (long long)blocks);
  ReArgs a{};
  a.cap = (int64_t)block_size * max_blocks;
  FCU_REQUIRE(a.cap <= 1 << 30, "fcu_cache_reorder: %lld slots per sequence (at most 2^30)", (long long)a.cap);
  int64_t most = 0;
  for (int i = 0; i < n_arrays; i++) {
    FCU_REQUIRE(arrays[i].base && ((uintptr_t)arrays[i].base & 15) == 0, "fcu_cache_reorder: array %d is null or not 16-byte aligned", i);
    FCU_REQUIRE(arrays[i].heads > 0 && arrays[i].heads <= 65535 && arrays[i].unit > 0 && arrays[i].unit % 4 == 0 &&
                    arrays[i].unit <= 1 << 24 && (int64_t)block_size * arrays[i].unit <= (int64_t)1 << 34,
                "fcu_cache_reorder: array %d of %lld heads, %lld bytes a slot", i, (long long)arrays[i].heads,
                (long long)arrays[i].unit);
    a.base[i] = (uint8_t *)arrays[i].base;
    a.heads[i] = arrays[i].heads;
    a.unit[i] = arrays[i].unit;
    const int64_t pieces = arrays[i].heads * max_blocks * (((int64_t)block_size * arrays[i].unit + 15) / 16);
    most = pieces > most ? pieces : most;
  }
  if (B == 0 || layers == 0 || n_arrays == 0 || W == 1) return FCU_OK;
  FCU_REQUIRE(parents && lens, "fcu_cache_reorder: null pointer");
  a.n_arrays = n_arrays;
  a.layers = layers;
  a.blocks = blocks;
  a.table = table;
  a.parents = parents;
  a.lens = lens;
  a.bs = block_size;
  a.mb = max_blocks;
  a.B = B;
  a.W = W;
  // CTAs over a (sequence, layer): up to eight waves of them in all, a thread then walks the rest
  const int64_t pairs = (int64_t)B * layers, fill = (8 * 16 * (int64_t)ctx->num_sms + pairs - 1) / pairs;
  int64_t gx = (most + kReThreads - 1) / kReThreads;
  gx = gx < fill ? gx : fill;
  const size_t smem = (size_t)W * kReThreads * 16;
  static bool set[64] = {false};
  if (!set[ctx->device & 63]) {
    FCU_CHECK_CUDA(cudaFuncSetAttribute(cache_reorder_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        kMaxW * kReThreads * 16));
    set[ctx->device & 63] = true;
  }
  FCU_CHECK_CUDA(launch_pdl(cache_reorder_kernel, dim3((unsigned)gx, B, (unsigned)layers), dim3(kReThreads), smem,
                            ctx->stream, a));
  note_launch();
  return FCU_OK;
}

}  // extern "C"
