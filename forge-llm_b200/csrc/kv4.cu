// The 4-bit KV cache (layout and grid: kv4.cuh, include/forgecu.h): RoPE and
// quantized writes, values read back, and eviction by accumulated attention
// weight.  Its attention is in kv4_attn.cu.
#include "kv4.cuh"

namespace fcu {
namespace kv4 {

int view(const char *who, const fcu_kv4 *in, int64_t B, bool need_values, Cache *out) {
  FCU_REQUIRE(in != nullptr, "%s: null cache", who);
  FCU_REQUIRE(in->dH >= 2 && in->dH <= kMaxDh && in->dH % 2 == 0, "%s: head dim %d (even, 2..%d)", who, in->dH, kMaxDh);
  FCU_REQUIRE(in->n_kv > 0 && in->n_kv <= 65535, "%s: %d kv heads", who, in->n_kv);
  FCU_REQUIRE(in->layers > 0 && in->blocks >= 0 && in->block_size > 0 && in->max_blocks > 0,
              "%s: bad cache geometry", who);
  const int64_t cap = (int64_t)in->max_blocks * in->block_size;
  FCU_REQUIRE(cap <= 1 << 30, "%s: %lld slots per sequence (at most 2^30)", who, (long long)cap);
  FCU_REQUIRE(in->table || B * in->max_blocks <= in->blocks, "%s: %lld sequences of %d blocks in a cache of %lld blocks",
              who, (long long)B, in->max_blocks, (long long)in->blocks);
  // row indexes, and a row's byte offset, stay far inside 64 bits
  FCU_REQUIRE(in->blocks <= (int64_t)1 << 40 && in->layers <= 1 << 20 &&
                  (double)in->layers * in->blocks * in->n_kv * in->block_size <= 1e15,
              "%s: the cache is too large", who);
  if (need_values) {
    FCU_REQUIRE(in->k && in->v && in->kg && in->vg, "%s: null cache array", who);
    FCU_REQUIRE((((uintptr_t)in->k | (uintptr_t)in->v) & 15) == 0, "%s: codes are not 16-byte aligned", who);
    FCU_REQUIRE((((uintptr_t)in->kg | (uintptr_t)in->vg | (uintptr_t)in->weight | (uintptr_t)in->pos |
                  (uintptr_t)in->table) & 3) == 0,
                "%s: a grid, weight, position or table array is not 4-byte aligned", who);
  }
  out->k = (uint8_t *)in->k;
  out->v = (uint8_t *)in->v;
  out->kg = (uint32_t *)in->kg;
  out->vg = (uint32_t *)in->vg;
  out->weight = in->weight;
  out->pos = in->pos;
  out->table = in->table;
  out->layers = in->layers;
  out->blocks = in->blocks;
  out->nKV = in->n_kv;
  out->dH = in->dH;
  out->rb = pad(in->dH) / 2;
  out->bs = in->block_size;
  out->mb = in->max_blocks;
  out->cap = cap;
  // the smallest 2^s >= bs; mul = floor(2^32 (2^s - bs) / bs) + 1 (Granlund and Montgomery's multiplier for division)
  out->div_shift = 0;
  while (((int64_t)1 << out->div_shift) < out->bs) out->div_shift++;
  out->div_mul = (uint32_t)(((((uint64_t)1 << out->div_shift) - out->bs) << 32) / out->bs + 1);
  return FCU_OK;
}

namespace {

// ------------------------------------------------------------------ put
constexpr int kPutThreads = 256;
constexpr int kPutTokens = 8;    // tokens of one CTA, which share the frequencies' pow

struct PutArgs {
  float *qkv;
  int64_t ld;
  const int32_t *positions, *slots;
  double theta;
  Cache c;
  int T, nH, tokens;   // tokens per CTA
  int vec;             // rows and heads start on 16 bytes
};

// G lanes hold one head, 8 consecutive elements (one word of codes) each.
template <int G>
__global__ void __launch_bounds__(kPutThreads) kv4_put_kernel(PutArgs a) {
  pdl_trigger();
  __shared__ double freq[kMaxDh / 2];
  __shared__ float2 cs[kPutTokens][kMaxDh / 2];
  const Cache &c = a.c;
  const int half = c.dH / 2, chunks = (a.T + a.tokens - 1) / a.tokens;
  const int64_t b = blockIdx.x / chunks;
  const int t0 = (blockIdx.x % chunks) * a.tokens;
  const int nt = min(a.tokens, a.T - t0);
  if (a.theta > 0)
    for (int i = threadIdx.x; i < half; i += kPutThreads) freq[i] = 1.0 / pow(a.theta, (double)(2 * i) / c.dH);
  pdl_wait();
  const int64_t pos0 = (int64_t)a.positions[b] + t0, slot0 = (int64_t)a.slots[b] + t0;
  if (a.theta > 0) {
    __syncthreads();
    for (int i = threadIdx.x; i < nt * half; i += kPutThreads) {
      const int t = i / half, e = i - t * half;
      double s, co;
      sincos((double)(pos0 + t) * freq[e], &s, &co);
      cs[t][e] = make_float2((float)co, (float)s);
    }
    __syncthreads();
  }
  const int heads = a.nH + 2 * c.nKV, items = nt * heads;
  const int li = threadIdx.x % G, e0 = li * 8;
  // every lane of a warp stays in the loop for the shuffles
  for (int i0 = threadIdx.x / G; i0 - (int)(threadIdx.x / G) < items; i0 += kPutThreads / G) {
    const bool on = i0 < items;
    const int t = on ? i0 / heads : 0, head = on ? i0 - t * heads : 0;
    const int64_t j = slot0 + t;
    int64_t row = -1;
    if (on && j >= 0 && j < c.cap && pos0 + t >= 0) row = row_of(c, b, head < a.nH ? 0 : (head - a.nH) % c.nKV, j);
    float *src = a.qkv + (b * a.T + t0 + t) * a.ld + (int64_t)head * c.dH + e0;
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; u++) x[u] = 0.f;
    if (row >= 0) {
      if (a.vec) {
#pragma unroll
        for (int u = 0; u < 8; u += 4)
          if (e0 + u < c.dH) {
            const float4 f = *reinterpret_cast<const float4 *>(src + u);
            x[u] = f.x, x[u + 1] = f.y, x[u + 2] = f.z, x[u + 3] = f.w;
          }
      } else {
#pragma unroll
        for (int u = 0; u < 8; u++)
          if (e0 + u < c.dH) x[u] = src[u];
      }
      if (a.theta > 0 && head < a.nH + c.nKV) {
#pragma unroll
        for (int u = 0; u < 8; u += 2)
          if (e0 + u < c.dH) {
            const float2 w = cs[t][(e0 + u) / 2];
            const double p = x[u], q = x[u + 1], co = w.x, s = w.y;
            x[u] = (float)(p * co - q * s);
            x[u + 1] = (float)(p * s + q * co);
          }
      }
    }
    if (row >= 0 && head < a.nH) {
      if (a.theta > 0) {
        if (a.vec) {
#pragma unroll
          for (int u = 0; u < 8; u += 4)
            if (e0 + u < c.dH) *reinterpret_cast<float4 *>(src + u) = make_float4(x[u], x[u + 1], x[u + 2], x[u + 3]);
        } else {
#pragma unroll
          for (int u = 0; u < 8; u++)
            if (e0 + u < c.dH) src[u] = x[u];
        }
      }
    }
    float lo = INFINITY, hi = -INFINITY;
    int bad = 0;
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (e0 + u < c.dH) {
        lo = fminf(lo, x[u]);
        hi = fmaxf(hi, x[u]);
        bad |= !(fabsf(x[u]) < 0x1p127f);
      }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      bad |= __shfl_xor_sync(0xffffffffu, bad, o);
    }
    if (row < 0 || head < a.nH) continue;
    const __nv_bfloat16 base_b = __float2bfloat16_rn(lo);
    const float base = __bfloat162float(base_b);
    double range = (double)hi - (double)base;
    range = range > 0 ? range : 0;
    const __nv_bfloat16 step_b = __float2bfloat16_rn((float)(range / 15.0));
    const float step = __bfloat162float(step_b);
    uint32_t word = 0;
    if (!bad && step > 0) {
      const float inv = 1.0f / step;
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (e0 + u < c.dH) {
          // The quotient in fp32 is within 4e-6 of the true one (at most 15.1
          // here), so its rounding is the true one's unless it is that near
          // a half; then, and where 1 / step left the normal range, divide in
          // double.
          const float d = x[u] - base, qf = d * inv, r = rintf(qf);
          int code = (int)fminf(fmaxf(r, 0.f), 15.f);
          if (!(fabsf(fabsf(qf - r) - 0.5f) > 1e-4f) || !(step > 1e-30f && step < 1e30f))
            code = (int)fmin(fmax(rint(((double)x[u] - (double)base) / (double)step), 0.0), 15.0);
          word |= (uint32_t)code << (4 * u);
        }
    }
    const uint32_t grid = bad ? kNanGrid
                              : (uint32_t)__bfloat16_as_ushort(step_b) | (uint32_t)__bfloat16_as_ushort(base_b) << 16;
    const bool is_v = head >= a.nH + c.nKV;
    if (4 * li < c.rb) reinterpret_cast<uint32_t *>((is_v ? c.v : c.k) + row * c.rb)[li] = word;
    if (li == 0) {
      (is_v ? c.vg : c.kg)[row] = grid;
      if (!is_v) {
        if (c.weight) c.weight[row] = 0.f;
        if (c.pos) c.pos[row] = (int32_t)(pos0 + t);
      }
    }
  }
}

// ------------------------------------------------------------------ values
constexpr int kValThreads = 256;

struct ValArgs {
  Cache c;
  const int32_t *start;
  int T, tokens, lanes_log;   // tokens per CTA; lanes of one row
  float *K, *V;
  int vec;
};

__global__ void __launch_bounds__(kValThreads) kv4_values_kernel(ValArgs a) {
  pdl_trigger();
  const Cache &c = a.c;
  const int chunks = (a.T + a.tokens - 1) / a.tokens;
  const int64_t b = blockIdx.x / chunks;
  const int t0 = (blockIdx.x % chunks) * a.tokens;
  const int nt = min(a.tokens, a.T - t0);
  pdl_wait();
  const int64_t s0 = (int64_t)a.start[b] + t0;
  const int items = (nt * c.nKV) << a.lanes_log, li = threadIdx.x & ((1 << a.lanes_log) - 1), e0 = 8 * li;
  for (int i = threadIdx.x; i < items; i += kValThreads) {
    const int r = i >> a.lanes_log, t = r / c.nKV, h = r - t * c.nKV;
    if (e0 >= c.dH) continue;
    const int64_t j = s0 + t;
    const int64_t row = j >= 0 && j < c.cap ? row_of(c, b, h, j) : -1;
    const int64_t o = (((int64_t)b * a.T + t0 + t) * c.nKV + h) * c.dH + e0;
#pragma unroll
    for (int w = 0; w < 2; w++) {
      float *out = w ? a.V : a.K;
      if (!out) continue;
      uint32_t word = 0, grid = kNanGrid;
      if (row >= 0) {
        word = reinterpret_cast<const uint32_t *>((w ? c.v : c.k) + row * c.rb)[li];
        grid = (w ? c.vg : c.kg)[row];
      }
      const float step = grid_step(grid), base = grid_base(grid);
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; u++) x[u] = base + step * (float)((word >> (4 * u)) & 15u);   // the product is exact
      if (a.vec) {
#pragma unroll
        for (int u = 0; u < 8; u += 4)
          if (e0 + u < c.dH) *reinterpret_cast<float4 *>(out + o + u) = make_float4(x[u], x[u + 1], x[u + 2], x[u + 3]);
      } else {
#pragma unroll
        for (int u = 0; u < 8; u++)
          if (e0 + u < c.dH) out[o + u] = x[u];
      }
    }
  }
}

// ------------------------------------------------------------------ evict
constexpr int kEvThreads = 1024;
constexpr int kEvBins = 2048;
constexpr int64_t kEvSmemSlots = 40 * 1024;   // keys of one head kept in shared memory

struct EvArgs {
  Cache c;
  const int32_t *lens;
  int B, budget, recent;
  int32_t *new_lens;
  uint32_t *work;   // keys [layers * B * nKV][cap] where they do not fit in shared memory
};

// Exclusive block scan of v over kEvThreads threads; total in *sum.
__device__ __forceinline__ uint32_t scan_excl(uint32_t v, uint32_t *warp_sums, uint32_t *sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();   // warp_sums may still be read from the previous scan
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint32_t w = warp_sums[lane];
  uint32_t incl = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  *sum = __shfl_sync(0xffffffffu, incl, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, incl - w, warp);
  return before + x - v;
}

// Keys order as the weights: larger weight, larger key; NaN 0 (below -inf's
// 0x007fffff), a protected slot 0xffffffff (above +inf's 0xff800000).
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.0f);   // -0 is 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA per (head, sequence, layer): the budget-th largest key by three
// histogram passes (11 + 11 + 10 bits) over keys in shared memory, then the
// freed slots and the slots that move, both in slot order, and the moves.
__global__ void __launch_bounds__(kEvThreads) kv4_evict_kernel(EvArgs a) {
  pdl_trigger();
  extern __shared__ __align__(16) uint32_t keys_sm[];
  __shared__ uint32_t hist[kEvBins];
  __shared__ uint32_t wsum[32];
  __shared__ int s_max;
  __shared__ uint32_t s_bin, s_need;
  const Cache &c = a.c;
  const int h = blockIdx.x % c.nKV;
  const int64_t r = blockIdx.x / c.nKV;
  const int b = (int)(r % a.B);
  const int64_t l = r / a.B;
  const int tid = threadIdx.x;
  if (tid == 0) s_max = INT_MIN;
  pdl_wait();
  const int64_t len = a.lens[b];
  const int n = (int)(len < 0 ? 0 : len > c.cap ? c.cap : len);
  // a block that the cache does not have: the sequence stays as it is
  int bad = 0;
  if (c.table)
    for (int64_t i = tid; i * c.bs < n; i += kEvThreads) bad |= block_of(c, b, i) < 0;
  bad = __syncthreads_or(bad);
  if (l == 0 && h == 0 && tid == 0) a.new_lens[b] = bad ? a.lens[b] : min(n, a.budget);
  if (bad || n <= a.budget) return;
  const int64_t lrow = l * c.blocks * c.nKV * c.bs;
  uint32_t *keys = a.work ? a.work + (int64_t)blockIdx.x * c.cap : keys_sm;
  int mx = INT_MIN;
  for (int j = tid; j < n; j += kEvThreads) mx = max(mx, c.pos[lrow + row_of(c, b, h, j)]);
  mx = __reduce_max_sync(0xffffffffu, mx);
  if ((tid & 31) == 0) atomicMax(&s_max, mx);
  __syncthreads();
  const int64_t newest = (int64_t)s_max - a.recent;
  for (int j = tid; j < n; j += kEvThreads) {
    const int64_t row = lrow + row_of(c, b, h, j);
    keys[j] = c.pos[row] > newest ? 0xffffffffu : weight_key(c.weight[row]);
  }
  uint32_t prefix = 0, mask = 0, need = a.budget, equal = 0;
  for (int pass = 0; pass < 3; pass++) {
    const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    for (int i = tid; i < kEvBins; i += kEvThreads) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += kEvThreads) {
      const uint32_t k = keys[j];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // bins from the largest down, two to a thread
    const int hi = (1 << bits) - 1 - 2 * tid;
    const uint32_t c0 = hi >= 0 ? hist[hi] : 0, c1 = hi >= 1 ? hist[hi - 1] : 0;
    uint32_t total;
    const uint32_t before = scan_excl(c0 + c1, wsum, &total);
    if (before < need && need <= before + c0) s_bin = hi, s_need = need - before;
    else if (before + c0 < need && need <= before + c0 + c1) s_bin = hi - 1, s_need = need - before - c0;
    __syncthreads();
    need = s_need;
    equal = hist[s_bin];
    prefix |= s_bin << shift;
    mask |= ((1u << bits) - 1) << shift;
    __syncthreads();
  }
  // kept: keys above the threshold, and of those equal to it the first `need`
  // slots.  Freed slots below the budget and kept ones past it are listed in
  // the key array itself: an entry's place is never past the slot it is for,
  // and a tile's keys are read before its entries are written.
  uint32_t holes = 0, movers = 0, eq_before = 0;
  for (int j0 = 0; j0 < n; j0 += kEvThreads) {
    const int j = j0 + tid;
    const uint32_t k = j < n ? keys[j] : 0;
    const bool eq = j < n && k == prefix;
    bool keep = j < n && (k > prefix || eq);
    uint32_t total;
    if (equal != need) {
      const uint32_t er = eq_before + scan_excl(eq, wsum, &total);
      if (eq) keep = er < need;
      eq_before += total;
    }
    const bool hole = j < a.budget && !keep, mover = j >= a.budget && keep;
    const uint32_t at = scan_excl((uint32_t)hole | (uint32_t)mover << 16, wsum, &total);
    if (hole) keys[holes + (at & 0xffffu)] = j;
    if (mover) keys[a.budget + movers + (at >> 16)] = j;
    holes += total & 0xffffu;
    movers += total >> 16;
  }
  __syncthreads();
  const int per = c.rb / 16, units = 2 * per + 1;
  const uint32_t work = holes * units;
  for (uint32_t i = tid; i < work; i += kEvThreads) {
    const uint32_t m = i / units, u = i - m * units;
    const int64_t dst = lrow + row_of(c, b, h, keys[m]), src = lrow + row_of(c, b, h, keys[a.budget + m]);
    if (u < (uint32_t)(2 * per)) {
      uint8_t *x = u < (uint32_t)per ? c.k : c.v;
      const int q = u < (uint32_t)per ? u : u - per;
      reinterpret_cast<uint4 *>(x + dst * c.rb)[q] = reinterpret_cast<const uint4 *>(x + src * c.rb)[q];
    } else {
      c.kg[dst] = c.kg[src];
      c.vg[dst] = c.vg[src];
      c.weight[dst] = c.weight[src];
      c.pos[dst] = c.pos[src];
    }
  }
}

}  // namespace
}  // namespace kv4
}  // namespace fcu

using namespace fcu;
using namespace fcu::kv4;

extern "C" {

int fcu_kv4_row_bytes(int dH) { return dH < 2 || dH > kMaxDh || dH % 2 ? -1 : pad(dH) / 2; }

int fcu_kv4_put(fcu_ctx *ctx, float *qkv, int64_t ld_qkv, int B, int T, int nH, double theta,
                const int32_t *positions, const int32_t *slots, const fcu_kv4 *cache) {
  FCU_CTX(ctx);
  FCU_REQUIRE(B >= 0 && T >= 0, "fcu_kv4_put: B=%d T=%d", B, T);
  PutArgs a{};
  int rc = view("fcu_kv4_put", cache, B, true, &a.c);
  if (rc) return rc;
  FCU_REQUIRE(nH >= 0 && nH <= 65535, "fcu_kv4_put: %d q heads", nH);
  FCU_REQUIRE(theta >= 0 && theta < 1e300, "fcu_kv4_put: theta %g", theta);
  FCU_REQUIRE(ld_qkv >= (int64_t)(nH + 2 * a.c.nKV) * a.c.dH, "fcu_kv4_put: row stride %lld too small",
              (long long)ld_qkv);
  if (B == 0 || T == 0) return FCU_OK;
  FCU_REQUIRE(qkv && positions && slots, "fcu_kv4_put: null pointer");
  a.qkv = qkv;
  a.ld = ld_qkv;
  a.positions = positions;
  a.slots = slots;
  a.theta = theta;
  a.T = T;
  a.nH = nH;
  a.tokens = T < kPutTokens ? 1 : kPutTokens;
  a.vec = ld_qkv % 4 == 0 && a.c.dH % 4 == 0 && ((uintptr_t)qkv & 15) == 0;
  const int64_t grid = (int64_t)B * ((T + a.tokens - 1) / a.tokens);
  FCU_REQUIRE(grid <= INT_MAX, "fcu_kv4_put: %d x %d tokens in one call", B, T);
  const int words = a.c.rb / 4;
  cudaError_t e;
  if (words <= 4) e = launch_pdl(kv4_put_kernel<4>, dim3(grid), dim3(kPutThreads), 0, ctx->stream, a);
  else if (words <= 8) e = launch_pdl(kv4_put_kernel<8>, dim3(grid), dim3(kPutThreads), 0, ctx->stream, a);
  else if (words <= 16) e = launch_pdl(kv4_put_kernel<16>, dim3(grid), dim3(kPutThreads), 0, ctx->stream, a);
  else e = launch_pdl(kv4_put_kernel<32>, dim3(grid), dim3(kPutThreads), 0, ctx->stream, a);
  FCU_CHECK_CUDA(e);
  note_launch();
  return FCU_OK;
}

int fcu_kv4_values(fcu_ctx *ctx, const fcu_kv4 *cache, const int32_t *start, int B, int T, float *K, float *V) {
  FCU_CTX(ctx);
  FCU_REQUIRE(B >= 0 && T >= 0, "fcu_kv4_values: B=%d T=%d", B, T);
  ValArgs a{};
  int rc = view("fcu_kv4_values", cache, B, true, &a.c);
  if (rc) return rc;
  if (B == 0 || T == 0 || (!K && !V)) return FCU_OK;
  FCU_REQUIRE(start != nullptr, "fcu_kv4_values: null pointer");
  a.start = start;
  a.T = T;
  a.K = K;
  a.V = V;
  a.vec = a.c.dH % 4 == 0 && (((uintptr_t)K | (uintptr_t)V) & 15) == 0;
  while ((1 << a.lanes_log) < a.c.rb / 4) a.lanes_log++;
  // about four rounds of a CTA's threads
  a.tokens = (4 * kValThreads >> a.lanes_log) / a.c.nKV;
  a.tokens = a.tokens < 1 ? 1 : a.tokens > T ? T : a.tokens;
  const int64_t grid = (int64_t)B * ((T + a.tokens - 1) / a.tokens);
  FCU_REQUIRE(grid <= INT_MAX, "fcu_kv4_values: %d x %d tokens in one call", B, T);
  FCU_CHECK_CUDA(launch_pdl(kv4_values_kernel, dim3(grid), dim3(kValThreads), 0, ctx->stream, a));
  note_launch();
  return FCU_OK;
}

int64_t fcu_kv4_evict_work(fcu_ctx *ctx, const fcu_kv4 *cache, int B) {
  Cache c;
  if (!ctx || B < 0 || view("fcu_kv4_evict_work", cache, B, false, &c)) return -1;
  return c.cap <= kEvSmemSlots ? 0 : c.layers * B * c.nKV * c.cap * 4;
}

int fcu_kv4_evict(fcu_ctx *ctx, const fcu_kv4 *cache, const int32_t *seq_lens, int B, int budget, int recent,
                  int32_t *new_lens, void *work, int64_t work_bytes) {
  FCU_CTX(ctx);
  FCU_REQUIRE(B >= 0, "fcu_kv4_evict: B=%d", B);
  EvArgs a{};
  int rc = view("fcu_kv4_evict", cache, B, true, &a.c);
  if (rc) return rc;
  FCU_REQUIRE(a.c.weight && a.c.pos, "fcu_kv4_evict: the cache keeps no weights and positions");
  FCU_REQUIRE(budget >= 1 && recent >= 0 && recent <= budget, "fcu_kv4_evict: budget %d, recent %d", budget, recent);
  FCU_REQUIRE(a.c.cap <= 1 << 26, "fcu_kv4_evict: %lld slots per sequence (at most 2^26)", (long long)a.c.cap);
  if (B == 0) return FCU_OK;
  FCU_REQUIRE(seq_lens && new_lens, "fcu_kv4_evict: null pointer");
  FCU_REQUIRE(new_lens + B <= seq_lens || seq_lens + B <= new_lens, "fcu_kv4_evict: new_lens overlaps seq_lens");
  const int64_t need = fcu_kv4_evict_work(ctx, cache, B);
  FCU_REQUIRE(need == 0 || (work && work_bytes >= need && ((uintptr_t)work & 3) == 0),
              "fcu_kv4_evict: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)need);
  const int64_t grid = a.c.layers * B * a.c.nKV;
  FCU_REQUIRE(grid <= INT_MAX, "fcu_kv4_evict: %lld heads in one call", (long long)grid);
  a.lens = seq_lens;
  a.B = B;
  a.budget = budget;
  a.recent = recent;
  a.new_lens = new_lens;
  a.work = need ? (uint32_t *)work : nullptr;
  static bool set[64] = {false};
  if (!set[ctx->device & 63]) {
    FCU_CHECK_CUDA(cudaFuncSetAttribute(kv4_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)(kEvSmemSlots * 4)));
    set[ctx->device & 63] = true;
  }
  FCU_CHECK_CUDA(launch_pdl(kv4_evict_kernel, dim3(grid), dim3(kEvThreads), need ? 0 : (size_t)a.c.cap * 4,
                            ctx->stream, a));
  note_launch();
  return FCU_OK;
}

}  // extern "C"
