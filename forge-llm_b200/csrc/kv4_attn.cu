// Attention of one new token per sequence over the 4-bit KV cache
// (fcu_kv4_attn; layout in kv4.cuh).
//
//   s_j = scale (step_j q.c_j + base_j sum q),  p = softmax(s)
//   o_e = sum_j p_j step_j c_je + sum_j p_j base_j
#include "kv4.cuh"

namespace fcu {
namespace kv4 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 256;    // slots per CTA

struct AttnArgs {
  const float *q;
  int64_t ld_q;
  Cache c;
  const int32_t *lens;
  int B, nH, splits;
  float scale;
  float *out;
  float *part_o;    // [B, nH, splits, dH]
  float *part_ml;   // [B, nH, splits, 2]
  float *scores;    // [B, nH, cap], kept where the cache keeps weights
};

__device__ __forceinline__ int64_t length(const AttnArgs &a, int b) {
  const int64_t n = a.lens[b];
  return n < 0 ? 0 : n > a.c.cap ? a.c.cap : n;
}

__global__ void __launch_bounds__(kThreads) kv4_attn_kernel(AttnArgs a) {
  pdl_trigger();
  extern __shared__ __align__(16) float sm[];
  const Cache &c = a.c;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = a.nH / c.nKV, dP = 2 * c.rb, words = c.rb / 4;
  float *q_s = sm;                         // [g][dP]
  float *s_s = q_s + g * dP;               // [g][kChunk]
  float *o_s = s_s + g * kChunk;           // [kWarps][dP]
  float *qs_s = o_s + kWarps * dP;         // [g]
  float *m_s = qs_s + g, *l_s = m_s + g;   // [g]
  __shared__ int64_t rows[kChunk];
  pdl_wait();
  const int64_t n = length(a, b), p0 = (int64_t)split * kChunk;
  if (p0 >= n && !(split == 0 && n == 0)) return;
  const int np = (int)min((int64_t)kChunk, n - p0);
  const int nsplit = (int)((n + kChunk - 1) / kChunk);
  for (int i = threadIdx.x; i < g * dP; i += kThreads) {
    const int hg = i / dP, e = i - hg * dP;
    q_s[i] = e < c.dH ? a.q[(int64_t)b * a.ld_q + (int64_t)(h * g + hg) * c.dH + e] : 0.f;
  }
  for (int j = threadIdx.x; j < np; j += kThreads) rows[j] = row_of(c, b, h, p0 + j);
  __syncthreads();
  for (int hg = warp; hg < g; hg += kWarps) {
    float s = 0.f;
    for (int e = lane; e < dP; e += 32) s += q_s[hg * dP + e];
    s = warp_sum(s);
    if (lane == 0) qs_s[hg] = s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < np * g; i += kThreads) {
    const int j = i / g, hg = i - j * g;
    const uint32_t grid = rows[j] >= 0 ? c.kg[rows[j]] : kNanGrid;
    float s = 0.f;
    if (rows[j] >= 0)
      for (int w = 0; w < words; w++) {
        const uint32_t x = reinterpret_cast<const uint32_t *>(c.k + rows[j] * c.rb)[w];
#pragma unroll
        for (int u = 0; u < 8; u++) s = fmaf(q_s[hg * dP + 8 * w + u], (float)((x >> (4 * u)) & 15u), s);
      }
    s_s[hg * kChunk + j] = (s * grid_step(grid) + qs_s[hg] * grid_base(grid)) * a.scale;
  }
  __syncthreads();
  for (int hg = warp; hg < g; hg += kWarps) {
    float m = -INFINITY, l = 0.f;
    for (int j = lane; j < np; j += 32) m = fmaxf(m, s_s[hg * kChunk + j]);
    m = warp_max(m);
    for (int j = lane; j < np; j += 32) {
      const float s = s_s[hg * kChunk + j], p = expf(s - m);
      if (a.scores) a.scores[((int64_t)b * a.nH + h * g + hg) * c.cap + p0 + j] = s;
      s_s[hg * kChunk + j] = p;
      l += p;
    }
    l = warp_sum(l);
    if (lane == 0) {
      m_s[hg] = m;
      l_s[hg] = l;
    }
  }
  __syncthreads();
  for (int hg = 0; hg < g; hg++) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (lane < words)
      for (int j = warp; j < np; j += kWarps) {
        const uint32_t grid = rows[j] >= 0 ? c.vg[rows[j]] : kNanGrid;
        const uint32_t x = rows[j] >= 0 ? reinterpret_cast<const uint32_t *>(c.v + rows[j] * c.rb)[lane] : 0;
        const float p = s_s[hg * kChunk + j], w = p * grid_step(grid), z = p * grid_base(grid);
#pragma unroll
        for (int u = 0; u < 8; u++) acc[u] += fmaf(w, (float)((x >> (4 * u)) & 15u), z);
      }
    if (lane < words)
#pragma unroll
      for (int u = 0; u < 8; u++) o_s[warp * dP + 8 * lane + u] = acc[u];
    __syncthreads();
    const int64_t bh = (int64_t)b * a.nH + h * g + hg;
    for (int e = threadIdx.x; e < c.dH; e += kThreads) {
      float o = 0.f;
      for (int w = 0; w < kWarps; w++) o += o_s[w * dP + e];
      if (nsplit <= 1 && !a.scores) a.out[bh * c.dH + e] = n > 0 ? o / l_s[hg] : 0.f;
      else a.part_o[(bh * a.splits + split) * c.dH + e] = o;
    }
    if ((nsplit > 1 || a.scores) && threadIdx.x == 0) {
      a.part_ml[(bh * a.splits + split) * 2] = m_s[hg];
      a.part_ml[(bh * a.splits + split) * 2 + 1] = l_s[hg];
    }
    __syncthreads();
  }
}

// Merges the chunks: out = sum_s o_s e^(m_s - M) / sum_s l_s e^(m_s - M).
__global__ void __launch_bounds__(128) kv4_attn_combine(AttnArgs a) {
  pdl_trigger();
  const int b = blockIdx.y;
  const int64_t bh = (int64_t)b * a.nH + blockIdx.x;
  pdl_wait();
  const int64_t n = length(a, b);
  const int nsplit = (int)((n + kChunk - 1) / kChunk);
  if (nsplit <= 1 && !a.scores) return;
  const float *ml = a.part_ml + bh * a.splits * 2;
  float M = -INFINITY, L = 0.f;
  for (int s = 0; s < nsplit; s++) M = fmaxf(M, ml[2 * s]);
  for (int s = 0; s < nsplit; s++) L += ml[2 * s + 1] * expf(ml[2 * s] - M);
  for (int e = threadIdx.x; e < a.c.dH; e += blockDim.x) {
    float o = 0.f;
    for (int s = 0; s < nsplit; s++) o += a.part_o[(bh * a.splits + s) * a.c.dH + e] * expf(ml[2 * s] - M);
    a.out[bh * a.c.dH + e] = n > 0 ? o / L : 0.f;
  }
}

// weight_j += sum over the group's q heads of p_j.
__global__ void __launch_bounds__(kChunk) kv4_attn_weights(AttnArgs a) {
  pdl_trigger();
  const Cache &c = a.c;
  const int h = blockIdx.y, b = blockIdx.z, g = a.nH / c.nKV;
  __shared__ float m_s[kMaxGroup], l_s[kMaxGroup];
  pdl_wait();
  const int64_t n = length(a, b), j = (int64_t)blockIdx.x * kChunk + threadIdx.x;
  if ((int64_t)blockIdx.x * kChunk >= n) return;
  const int nsplit = (int)((n + kChunk - 1) / kChunk);
  if (threadIdx.x < g) {
    const float *ml = a.part_ml + ((int64_t)b * a.nH + h * g + threadIdx.x) * a.splits * 2;
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < nsplit; s++) M = fmaxf(M, ml[2 * s]);
    for (int s = 0; s < nsplit; s++) L += ml[2 * s + 1] * expf(ml[2 * s] - M);
    m_s[threadIdx.x] = M;
    l_s[threadIdx.x] = L;
  }
  __syncthreads();
  if (j >= n) return;
  const int64_t row = row_of(c, b, h, j);
  if (row < 0) return;
  float w = 0.f;
  for (int hg = 0; hg < g; hg++)
    w += expf(a.scores[((int64_t)b * a.nH + h * g + hg) * c.cap + j] - m_s[hg]) / l_s[hg];
  c.weight[row] += w;
}

// Floats of workspace: part_o, part_ml, and the scores where weights are kept.
int64_t work_floats(const Cache &c, int B, int nH, int splits) {
  const int64_t bh = (int64_t)B * nH;
  return (splits > 1 || c.weight ? bh * splits * (c.dH + 2) : 0) + (c.weight ? bh * c.cap : 0);
}

int checked(const char *who, const fcu_kv4 *cache, int B, int nH, bool arrays, Cache *c) {
  FCU_REQUIRE(B >= 0 && B <= 65535, "%s: B=%d", who, B);
  int rc = view(who, cache, B, arrays, c);
  if (rc) return rc;
  FCU_REQUIRE(nH > 0 && nH % c->nKV == 0 && nH / c->nKV <= kMaxGroup, "%s: %d q heads on %d kv heads", who, nH, c->nKV);
  return FCU_OK;
}

}  // namespace
}  // namespace kv4
}  // namespace fcu

using namespace fcu;
using namespace fcu::kv4;

extern "C" {

int64_t fcu_kv4_attn_work(fcu_ctx *ctx, const fcu_kv4 *cache, int B, int nH) {
  Cache c;
  if (!ctx || checked("fcu_kv4_attn_work", cache, B, nH, false, &c)) return -1;
  return 4 * work_floats(c, B, nH, div_up(c.cap, kChunk));
}

int fcu_kv4_attn(fcu_ctx *ctx, const float *q, int64_t ld_q, const fcu_kv4 *cache, const int32_t *seq_lens, int B,
                 int nH, double scale, float *out, void *work, int64_t work_bytes) {
  FCU_CTX(ctx);
  AttnArgs a{};
  int rc = checked("fcu_kv4_attn", cache, B, nH, true, &a.c);
  if (rc) return rc;
  FCU_REQUIRE(ld_q >= (int64_t)nH * a.c.dH, "fcu_kv4_attn: q row stride %lld too small", (long long)ld_q);
  if (B == 0) return FCU_OK;
  FCU_REQUIRE(q && seq_lens && out, "fcu_kv4_attn: null pointer");
  a.q = q;
  a.ld_q = ld_q;
  a.lens = seq_lens;
  a.B = B;
  a.nH = nH;
  a.scale = (float)scale;
  a.out = out;
  a.splits = div_up(a.c.cap, kChunk);
  const int64_t need = 4 * work_floats(a.c, B, nH, a.splits);
  FCU_REQUIRE(need == 0 || (work && work_bytes >= need && ((uintptr_t)work & 15) == 0),
              "fcu_kv4_attn: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)need);
  const int64_t bh = (int64_t)B * nH;
  a.part_o = (float *)work;
  a.part_ml = a.part_o + bh * a.splits * a.c.dH;
  a.scores = a.c.weight ? a.part_ml + bh * a.splits * 2 : nullptr;
  const int g = nH / a.c.nKV, dP = 2 * a.c.rb;
  const size_t smem = sizeof(float) * ((size_t)g * dP + (size_t)g * kChunk + kWarps * dP + 3 * g);
  static bool set[64] = {false};
  if (!set[ctx->device & 63]) {
    FCU_CHECK_CUDA(cudaFuncSetAttribute(kv4_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024));
    set[ctx->device & 63] = true;
  }
  FCU_CHECK_CUDA(launch_pdl(kv4_attn_kernel, dim3(a.splits, a.c.nKV, B), dim3(kThreads), smem, ctx->stream, a));
  note_launch();
  if (a.splits > 1 || a.scores) {
    FCU_CHECK_CUDA(launch_pdl(kv4_attn_combine, dim3(nH, B), dim3(128), 0, ctx->stream, a));
    note_launch();
  }
  if (a.scores) {
    FCU_CHECK_CUDA(launch_pdl(kv4_attn_weights, dim3(a.splits, a.c.nKV, B), dim3(kChunk), 0, ctx->stream, a));
    note_launch();
  }
  return FCU_OK;
}

}  // extern "C"
