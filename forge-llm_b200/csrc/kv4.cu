// The 4-bit KV cache (layout and grid: kv4.cuh, include/forgecu.h): RoPE and
// quantized writes, values read back, and eviction by accumulated attention
// weight.  Its attention is in kv4_attn.cu.
#include <string.h>

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
  FCU_REQUIRE(in->table || B * in->max_blocks <= in->blocks,
              "%s: %lld sequences of %d blocks in a cache of %lld blocks", who, (long long)B, in->max_blocks, (long long)in->blocks);
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
// A CTA takes up to kPutTokens tokens of one sequence: the frequencies once, the
// tokens' cosines and sines, then q (four elements to a thread, the same ones of
// every token) and k and v (eight to a lane, a code word).  Bound by HBM for a
// prompt's tokens (q both ways, k and v in): 4 x 2048 tokens, 32 / 8 heads of 128,
// 76 us = 4.7 TB/s of 355 MB, with issue 61 % busy; by latency for one token
// (32 sequences: 6 us, most of it the pow and sincos of one warp).
constexpr int kPutThreads = 256;
constexpr int kPutTokens = 8;    // share the frequencies' pow
constexpr int kPutBatch = 4;     // 16-byte loads of q that a thread has in flight

struct PutArgs {
  float *qkv;
  int64_t ld;
  const int32_t *positions, *slots;
  double theta;
  Cache c;
  int T, nH, tokens;   // tokens per CTA
  int vec;             // rows and heads start on 16 bytes
};

// The rotation of neighbouring pairs by angles whose (cos, sin) are given, as a
// rotation in double rounds to fp32.  The products' and the sum's errors are
// carried along in fp32, about 2^-46 of the result in all, so that the roundings
// agree but for results that near a tie (conversions to and from fp64 run at a
// sixteenth of the rate and took a third of a prompt chunk's time); values that
// leave fp32's normal range on the way take doubles.
__device__ __forceinline__ float diff_of_products(float a, float b, float c, float d) {
  const float p = a * b, pe = fmaf(a, b, -p), q = c * d, qe = fmaf(c, d, -q);
  const float s = p - q, z = s - p, e = (p - (s - z)) - (q + z);
  return s + (e + (pe - qe));
}
template <int N>
__device__ __forceinline__ void rotate(float (&x)[N], const float2 (&w)[N / 2]) {
  float lo = INFINITY, hi = 0.f;
#pragma unroll
  for (int u = 0; u < N; u += 2) {
    const float m = fmaxf(fabsf(x[u]), fabsf(x[u + 1]));
    lo = fminf(lo, m);
    hi = fmaxf(hi, m);
  }
  float y[N], sum = 0.f;
#pragma unroll
  for (int u = 0; u < N; u += 2) {
    y[u] = diff_of_products(x[u], w[u / 2].x, x[u + 1], w[u / 2].y);
    y[u + 1] = diff_of_products(x[u], w[u / 2].y, -x[u + 1], w[u / 2].x);
    sum += y[u] + y[u + 1];
  }
  if (!(lo > 0x1p-60f && hi < 0x1p120f && sum == sum)) {
#pragma unroll
    for (int u = 0; u < N; u += 2) {
      const double p = x[u], q = x[u + 1], co = w[u / 2].x, s = w[u / 2].y;
      y[u] = (float)(p * co - q * s);
      y[u + 1] = (float)(p * s + q * co);
    }
  }
#pragma unroll
  for (int u = 0; u < N; u++) x[u] = y[u];
}

// FULL: a head has no padding (dH == 32 W).
template <int W, bool FULL>
__global__ void __launch_bounds__(kPutThreads, 4) kv4_put_kernel(PutArgs a) {
  pdl_trigger();
  __shared__ double freq[16 * W];
  __shared__ float2 cs[kPutTokens][16 * W];
  __shared__ int64_t row_s[kPutTokens];      // head 0's row of each token's slot; -1: the token changes nothing
  const Cache &c = a.c;
  const int dH = FULL ? 32 * W : c.dH, half = dH / 2, chunks = (a.T + a.tokens - 1) / a.tokens, tid = threadIdx.x;
  const int64_t b = blockIdx.x / chunks;
  const int t0 = (blockIdx.x % chunks) * a.tokens;
  const int nt = min(a.tokens, a.T - t0);
  if (a.theta > 0)
    for (int i = tid; i < half; i += kPutThreads) freq[i] = 1.0 / pow(a.theta, (double)(2 * i) / dH);
  pdl_wait();
  const int64_t pos0 = (int64_t)a.positions[b] + t0, slot0 = (int64_t)a.slots[b] + t0;
  if (tid < nt) {
    const int64_t j = slot0 + tid;
    row_s[tid] = j >= 0 && j < c.cap && pos0 + tid >= 0 && pos0 + tid <= INT_MAX ? row_of(c, b, 0, j) : -1;
  }
  __syncthreads();
  float *x0 = a.qkv + (b * a.T + t0) * a.ld;
  if (a.theta > 0) {
    for (int i = tid; i < nt * half; i += kPutThreads) {
      const int t = i / half, e = i - t * half;
      double s, co;
      sincos((double)(pos0 + t) * freq[e], &s, &co);
      cs[t][e] = make_float2((float)co, (float)s);
    }
    __syncthreads();
    // q, four elements to a thread, the same ones of every token
    if (a.vec) {
      for (int i = tid; i < a.nH * (8 * W); i += kPutThreads) {
        const int h = i / (8 * W), e = 4 * (i - h * 8 * W);
        if (e >= dH) continue;
        float *p = x0 + h * dH + e;
        for (int t1 = 0; t1 < nt; t1 += kPutBatch) {
          float4 x[kPutBatch];
#pragma unroll
          for (int k = 0; k < kPutBatch; k++)
            if (t1 + k < nt && row_s[t1 + k] >= 0) x[k] = *reinterpret_cast<const float4 *>(p + (t1 + k) * a.ld);
#pragma unroll
          for (int k = 0; k < kPutBatch; k++)
            if (t1 + k < nt && row_s[t1 + k] >= 0) {
              const float2 w[2] = {cs[t1 + k][e / 2], cs[t1 + k][e / 2 + 1]};
              float y[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
              rotate(y, w);
              *reinterpret_cast<float4 *>(p + (t1 + k) * a.ld) = make_float4(y[0], y[1], y[2], y[3]);
            }
        }
      }
    } else {
      for (int i = tid; i < nt * a.nH * half; i += kPutThreads) {
        const int th = i / half, e = i - th * half, t = th / a.nH, h = th - t * a.nH;
        if (row_s[t] < 0) continue;
        float *p = x0 + t * a.ld + (int64_t)h * dH + 2 * e, y[2] = {p[0], p[1]};
        const float2 w[1] = {cs[t][e]};
        rotate(y, w);
        p[0] = y[0];
        p[1] = y[1];
      }
    }
  }
  // k and v: G lanes hold one head of a token, eight consecutive elements (one
  // word of codes) each; every lane of a warp stays in the loops for the shuffles
  constexpr int G = W == 1 ? 4 : W == 2 ? 8 : W <= 4 ? 16 : 32;
  const int heads = 2 * c.nKV, li = tid % G, e0 = li * 8;
  for (int h0 = tid / G; h0 - tid / G < heads; h0 += kPutThreads / G) {
    const bool on = h0 < heads, is_v = h0 >= c.nKV;
    const float *src = x0 + (int64_t)(a.nH + h0) * dH + e0;
    uint8_t *codes = is_v ? c.v : c.k;
    uint32_t *grids = is_v ? c.vg : c.kg;
    const int64_t head = (int64_t)(is_v ? h0 - c.nKV : h0) * c.bs;
    for (int t = 0; t < nt; t++, src += a.ld) {
      const int64_t row = on && row_s[t] >= 0 ? row_s[t] + head : -1;
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; u++) x[u] = 0.f;
      if (row >= 0) {
        if (a.vec) {
#pragma unroll
          for (int u = 0; u < 8; u += 4)
            if (e0 + u < dH) {
              const float4 f = *reinterpret_cast<const float4 *>(src + u);
              x[u] = f.x, x[u + 1] = f.y, x[u + 2] = f.z, x[u + 3] = f.w;
            }
        } else {
#pragma unroll
          for (int u = 0; u < 8; u++)
            if (e0 + u < dH) x[u] = src[u];
        }
        if (a.theta > 0 && !is_v) {
          if (e0 + 8 <= dH) {
            const float2 w[4] = {cs[t][e0 / 2], cs[t][e0 / 2 + 1], cs[t][e0 / 2 + 2], cs[t][e0 / 2 + 3]};
            rotate(x, w);
          } else {
#pragma unroll
            for (int u = 0; u < 8; u += 2)
              if (e0 + u < dH) {
                float y[2] = {x[u], x[u + 1]};
                const float2 w[1] = {cs[t][(e0 + u) / 2]};
                rotate(y, w);
                x[u] = y[0];
                x[u + 1] = y[1];
              }
          }
        }
      }
      float lo = INFINITY, hi = -INFINITY;
      bool bad = false;
#pragma unroll
      for (int u = 0; u < 8; u++)
        if (e0 + u < dH) {
          lo = fminf(lo, x[u]);
          hi = fmaxf(hi, x[u]);
          bad |= x[u] != x[u];
        }
      if (bad) lo = -INFINITY;                      // (fminf passes a NaN over)
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      if (row < 0) continue;
      bad = !(lo > -0x1p127f && hi < 0x1p127f);
      const __nv_bfloat16 base_b = __float2bfloat16_rn(lo);
      const float base = __bfloat162float(base_b);
      // step = bf16(fp32((hi - base) / 15)): the product below is within 4 units
      // of its last place of that fp32 value, so it rounds to the same bf16 unless
      // it is that near the middle of two (or hi - base near the ends of fp32)
      float q15 = fmaxf(hi - base, 0.f) * (1.0f / 15.0f);
      if (abs((int)(__float_as_uint(q15) & 0xffffu) - 0x8000) <= 16 || !(q15 >= 1e-30f && q15 < 0x1p123f)) {
        const double range = (double)hi - (double)base;
        q15 = (float)((range > 0 ? range : 0.0) / 15.0);
      }
      const __nv_bfloat16 step_b = __float2bfloat16_rn(q15);
      const float step = __bfloat162float(step_b);
      uint32_t word = 0;
      if (!bad && step > 0) {
        // The quotient in fp32 is within 4e-6 of the true one (at most 15.1 here),
        // so its rounding is the true one's unless it is that near a half; then,
        // and where 1 / step left the normal range, divide in double.
        const float inv = 1.0f / step;
        float near = 1.f;
#pragma unroll
        for (int u = 0; u < 8; u++) {
          const float q = fminf(fmaxf((x[u] - base) * inv, 0.f), 15.f);
          const float m = q + 0x1.8p23f;      // q rounded, ties to even
          near = fminf(near, fabsf(fabsf(q - (m - 0x1.8p23f)) - 0.5f));
          if (e0 + u < dH) word |= (__float_as_uint(m) & 15u) << (4 * u);
        }
        if (!(near > 1e-4f) || !(step > 1e-30f && step < 1e30f)) {
          word = 0;
#pragma unroll
          for (int u = 0; u < 8; u++)
            if (e0 + u < dH)
              word |= (uint32_t)fmin(fmax(rint(((double)x[u] - (double)base) / (double)step), 0.0), 15.0) << (4 * u);
        }
      }
      const uint32_t grid = bad ? kNanGrid
                                : (uint32_t)__bfloat16_as_ushort(step_b) | (uint32_t)__bfloat16_as_ushort(base_b) << 16;
      if (4 * li < c.rb) reinterpret_cast<uint32_t *>(codes + row * c.rb)[li] = word;
      if (li == 0) {
        grids[row] = grid;
        if (!is_v) {
          if (c.weight) c.weight[row] = 0.f;
          if (c.pos) c.pos[row] = (int32_t)(pos0 + t);
        }
      }
    }
  }
}

// ------------------------------------------------------------------ values
// Four elements to a thread, one 16-byte store each of K and V.  Bound by HBM
// (the values written): 4 x 2048 slots of 8 heads of 128, 16 us = 4.7 TB/s.
constexpr int kValThreads = 256;
constexpr int kValBatch = 4;
constexpr int kValTokens = 8;    // slots of a CTA

struct ValArgs {
  Cache c;
  const int32_t *start;
  int T;
  float *K, *V;
  int vec;
};

template <int W>
__global__ void __launch_bounds__(kValThreads) kv4_values_kernel(ValArgs a) {
  pdl_trigger();
  __shared__ int64_t row_s[kValTokens];      // head 0's row of each slot; -1: there is none
  const Cache &c = a.c;
  const int chunks = (a.T + kValTokens - 1) / kValTokens;
  const int64_t b = blockIdx.x / chunks;
  const int t0 = (blockIdx.x % chunks) * kValTokens;
  const int nt = min(kValTokens, a.T - t0);
  pdl_wait();
  if (threadIdx.x < nt) {
    const int64_t j = (int64_t)a.start[b] + t0 + threadIdx.x;
    row_s[threadIdx.x] = j >= 0 && j < c.cap ? row_of(c, b, 0, j) : -1;
  }
  __syncthreads();
  const int kvd = c.nKV * c.dH;
  // four elements to a thread, the same ones of every slot
  for (int i = threadIdx.x; i < c.nKV * (8 * W); i += kValThreads) {
    const int h = i / (8 * W), e = 4 * (i - h * 8 * W);
    if (e >= c.dH) continue;
    const int64_t o = (b * a.T + t0) * kvd + h * c.dH + e;
    for (int t1 = 0; t1 < nt; t1 += kValBatch) {
      uint32_t code[kValBatch][2], grid[kValBatch][2];
#pragma unroll
      for (int k = 0; k < kValBatch; k++) {
        const int64_t row = t1 + k < nt && row_s[t1 + k] >= 0 ? row_s[t1 + k] + (int64_t)h * c.bs : -1;
        code[k][0] = code[k][1] = 0;
        grid[k][0] = grid[k][1] = kNanGrid;
        if (row >= 0) {
          code[k][0] = reinterpret_cast<const uint16_t *>(c.k + row * c.rb)[e / 4];
          code[k][1] = reinterpret_cast<const uint16_t *>(c.v + row * c.rb)[e / 4];
          grid[k][0] = c.kg[row];
          grid[k][1] = c.vg[row];
        }
      }
#pragma unroll
      for (int k = 0; k < kValBatch; k++)
#pragma unroll
        for (int w = 0; w < 2; w++) {
          float *out = w ? a.V : a.K;
          if (t1 + k >= nt || !out) continue;
          out += o + (int64_t)(t1 + k) * kvd;
          const float step = grid_step(grid[k][w]), base = grid_base(grid[k][w]);
          float x[4];
#pragma unroll
          for (int u = 0; u < 4; u++) {
            const float code_f = __uint_as_float(((code[k][w] >> (4 * u)) & 15u) | 0x4b000000u) - 0x1p23f;
            x[u] = base + step * code_f;                  // the product is exact
          }
          if (a.vec) {
            *reinterpret_cast<float4 *>(out) = make_float4(x[0], x[1], x[2], x[3]);
          } else {
#pragma unroll
            for (int u = 0; u < 4; u++)
              if (e + u < c.dH) out[u] = x[u];
          }
        }
    }
  }
}

// ------------------------------------------------------------------ evict
constexpr int kEvThreads = 512;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvBins = 2048;
constexpr int kEvBatch = 2;                   // loads of a thread in flight, of four slots each where they line up
constexpr int kEvPieces = 4;
// Moves of one head that the selecting CTA makes itself.  Calls on 384 heads of 64 cut in
// half, moves here and in kv4_move_kernel: 300 moves 9.7 and 12.5 us, 500 10.7 and 13.3,
// 1000 13.5 and 17.2, 2000 17.3 and 23.0 (32 heads of 128, 1000 moves: 8.5 and 10.9).
// kv4_move_kernel was taken for 512 heads of 128 with 2000 moves each, where a CTA's moves
// wait for its selection; the limit has room below that.
constexpr int kEvInline = 512;
// Keys that are ranked directly, one to a thread at most (64 in place of 512: 512 heads cut
// from 16001 to 2048 slots 52.9 us, so 51.5; from 4001 to 1000 25.5 and 25.1).
constexpr int kEvFew = kEvThreads;
constexpr int kEvSmemSlots = 40 * 1024;   // keys of one head kept in shared memory

struct EvArgs {
  Cache c;
  const int32_t *lens;
  int B, budget, recent;
  int32_t *new_lens;
  uint32_t *keys;   // [heads][padded cap] where they do not fit in shared memory (heads: layers * B * nKV)
  // for kv4_move_kernel, where a head may have more moves than kEvInline: their
  // number, and slots to and from [heads][most]
  uint32_t *count;
  int32_t *to, *from;
  int most;
};

// Keys are kept with a word of padding after every 32, so that threads that walk
// neighbouring runs of slots meet different banks.
__host__ __device__ inline int ev_at(int j) { return j + (j >> 5); }   // (j at most 2^26)

// Exclusive block scan of v; total in *sum.
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
  const uint32_t w = lane < kEvWarps ? warp_sums[lane] : 0;
  uint32_t incl = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  *sum = __shfl_sync(0xffffffffu, incl, 31);
  return __shfl_sync(0xffffffffu, incl - w, warp) + x - v;
}

// Keys order as the weights: larger weight, larger key; NaN 0 (below -inf's
// 0x007fffff), a protected slot 0xffffffff (above +inf's 0xff800000).
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.0f);   // -0 is 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// G neighbouring values, or `other`.
template <int G, typename T>
__device__ __forceinline__ void load_slots(T (&x)[G], const T *p, bool on, T other) {
  if constexpr (G == 4) {
    static_assert(sizeof(T) == 4, "");
    const int4 v = on ? *reinterpret_cast<const int4 *>(p) : int4{0, 0, 0, 0};
    const int y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      T f;
      memcpy(&f, &y[e], 4);
      x[e] = on ? f : other;
    }
  } else {
    x[0] = on ? *p : other;
  }
}

// One CTA per (head, sequence, layer).  The budget-th largest key is found by
// histograms over the range that the keys span: 2048 bins of equal width, then
// the bin that holds it again, until its keys are few enough to be ranked one
// against the other (weights spread over many magnitudes; bins of the range
// itself meet fewer collisions than bins of leading bits).  Then the freed slots
// and the slots that move are listed, both in slot order, and moved.  Instruction
// bound (issue 57 % busy): 4 x 16 x 8 heads of 16001 slots, 45 us for 67 MB of
// weights and positions.
// VEC: four slots of a head are 16 aligned bytes of weight and pos.  CTAS:
// resident per SM, by registers: 3 while a head's keys are short, since then a
// few hundred heads run at once (12 x 8 x 4 heads of 1025 slots 9.3 us, 11.7 with 2; of
// 8000, 17.6 and 20.5; 4 x 16 x 8 heads of 8000 24.7 and 25.6); with long ones shared
// memory leaves no more anyway and the registers are worth more (4 x 16 x 8 heads of
// 16001 slots cut to 2048, before the moves had a kernel: 155 us, 177 with 3).
template <bool SMEM, bool VEC, int CTAS>
__global__ void __launch_bounds__(kEvThreads, CTAS) kv4_evict_kernel(EvArgs a) {
  pdl_trigger();
  extern __shared__ __align__(16) uint32_t keys_sm[];
  __shared__ uint32_t hist[kEvBins];
  __shared__ uint32_t wsum[32];
  __shared__ int s_max, s_n;
  __shared__ uint32_t s_lo, s_hi, s_bin, s_need, s_few;
  const Cache &c = a.c;
  const int h = blockIdx.x % c.nKV;
  const int64_t r = blockIdx.x / c.nKV;
  const int b = (int)(r % a.B);
  const int64_t l = r / a.B;
  const int tid = threadIdx.x, lane = tid & 31;
  constexpr int G = VEC ? 4 : 1;
  pdl_wait();
  if (tid == 0) {
    s_max = INT_MIN, s_lo = 0xffffffffu, s_hi = 0, s_few = 0;
    const int64_t len = a.lens[b];
    s_n = (int)(len < 0 ? 0 : len > c.cap ? c.cap : len);      // one reader, so that the threads agree
  }
  __syncthreads();
  const int n = s_n;
  const int64_t lrow = l * c.blocks * c.nKV * c.bs;
  const bool cut = n > a.budget;
  uint32_t *keys = SMEM ? keys_sm : a.keys + (int64_t)blockIdx.x * ev_at((int)c.cap);
  // the row of slot 0 where all slots lie in one block
  int64_t flat = -1;
  if (c.mb == 1) {
    flat = block_of(c, b, 0);
    if (flat >= 0) flat = (flat * c.nKV + h) * c.bs;
  }
  // the newest position; a block that the cache does not have leaves the sequence
  // as it is
  int bad = c.mb == 1 && flat < 0 && n > 0, mx = INT_MIN;
  if (cut || (l == 0 && h == 0 && c.table)) {
    for (int j0 = G * tid; j0 < n; j0 += 2 * kEvBatch * G * kEvThreads) {
      int p[2 * kEvBatch][G];
#pragma unroll
      for (int i = 0; i < 2 * kEvBatch; i++) {
        const int j = j0 + i * G * kEvThreads;
        const int64_t at = j >= n ? -2 : flat >= 0 ? flat + j : row_of(c, b, h, j);
        bad |= at == -1;
        load_slots<G>(p[i], c.pos + lrow + at, cut && at >= 0, INT_MIN);
      }
#pragma unroll
      for (int i = 0; i < 2 * kEvBatch; i++)
#pragma unroll
        for (int e = 0; e < G; e++)
          if (j0 + i * G * kEvThreads + e < n) mx = max(mx, p[i][e]);
    }
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (lane == 0) atomicMax(&s_max, mx);
    bad = __syncthreads_or(bad);
  }
  if (a.most && tid == 0 && (bad || !cut)) a.count[blockIdx.x] = 0;
  if (l == 0 && h == 0 && tid == 0) a.new_lens[b] = bad ? n : min(n, a.budget);
  if (bad || !cut) return;
  // positions from `fresh` on are protected (none if there are no recent ones)
  const int64_t first = (int64_t)s_max - a.recent + 1;
  const int fresh = first < INT_MIN ? INT_MIN : first > INT_MAX ? INT_MAX : (int)first;
  const bool some = a.recent > 0;
  uint32_t lo = 0xffffffffu, hi = 0, safe = 0;      // the other slots' range; the protected ones
  for (int j0 = G * tid; j0 < n; j0 += kEvBatch * G * kEvThreads) {
    float w[kEvBatch][G];
    int p[kEvBatch][G];
#pragma unroll
    for (int i = 0; i < kEvBatch; i++) {
      const int j = j0 + i * G * kEvThreads;
      const int64_t at = j >= n ? 0 : flat >= 0 ? flat + j : row_of(c, b, h, j);
      load_slots<G>(w[i], c.weight + lrow + at, j < n, 0.f);
      load_slots<G>(p[i], c.pos + lrow + at, j < n, 0);
    }
#pragma unroll
    for (int i = 0; i < kEvBatch; i++) {
      const int j = j0 + i * G * kEvThreads;
      uint32_t *dst = keys + ev_at(j);              // (four slots do not cross a word of padding)
#pragma unroll
      for (int e = 0; e < G; e++)
        if (j + e < n) {
          uint32_t k = weight_key(w[i][e]);
          if (some && p[i][e] >= fresh) {
            k = 0xffffffffu;
            safe++;
          } else {
            lo = min(lo, k);
            hi = max(hi, k);
          }
          dst[e] = k;
        }
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) {
    atomicMin(&s_lo, lo);
    atomicMax(&s_hi, hi);
  }
  uint32_t protect;
  scan_excl(safe, wsum, &protect);                  // (its barriers cover s_lo and s_hi)
  lo = s_lo;
  hi = s_hi;
  // the threshold: keys above it stay, and `need` of the `equal` keys that are it
  uint32_t prefix = 0xffffffffu, need = a.budget, equal = protect;
  if (protect < (uint32_t)a.budget) {
    need -= protect;                                // of the keys in [lo, hi]
    while (true) {
      const uint32_t span = hi - lo;
      const int shift = span < kEvBins ? 0 : 21 - __clz(span);   // span >> shift < kEvBins
      for (int i = tid; i < kEvBins; i += kEvThreads) hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int j = tid; j < n; j += kEvThreads) {
        const uint32_t k = keys[ev_at(j)] - lo;
        if (k <= span) atomicAdd(&hist[k >> shift], 1u);
      }
      __syncthreads();
      // bins from the largest down, four to a thread
      uint32_t cnt[kEvBins / kEvThreads], sum = 0, total;
#pragma unroll
      for (int i = 0; i < kEvBins / kEvThreads; i++) {
        cnt[i] = hist[kEvBins - 1 - (kEvBins / kEvThreads * tid + i)];
        sum += cnt[i];
      }
      uint32_t before = scan_excl(sum, wsum, &total);
#pragma unroll
      for (int i = 0; i < kEvBins / kEvThreads; i++) {
        if (before < need && need <= before + cnt[i]) {
          s_bin = kEvBins - 1 - (kEvBins / kEvThreads * tid + i);
          s_need = need - before;
        }
        before += cnt[i];
      }
      __syncthreads();
      need = s_need;
      equal = hist[s_bin];
      lo += s_bin << shift;
      hi = min(hi, lo + ((1u << shift) - 1));
      prefix = lo;
      __syncthreads();
      if (shift == 0) break;
      if (equal <= kEvFew) {
        // the bin's keys, each ranked against the others; equal ones share a rank
        for (int j = tid; j < n; j += kEvThreads) {
          const uint32_t k = keys[ev_at(j)];
          if (k - lo <= hi - lo) hist[atomicAdd(&s_few, 1u)] = k;
        }
        __syncthreads();
        if (tid < (int)equal) {
          const uint32_t k = hist[tid];
          uint32_t above = 0, same = 0;
          for (uint32_t i = 0; i < equal; i++) {
            above += hist[i] > k;
            same += hist[i] == k;
          }
          if (above < need && need <= above + same) {   // (by every thread that holds this key)
            s_lo = k;
            s_need = need - above;
            s_bin = same;
          }
        }
        __syncthreads();
        prefix = s_lo;
        need = s_need;
        equal = s_bin;
        break;
      }
    }
  }
  // kept: keys above the threshold, and of those equal to it the first `need`
  // slots.  A thread takes a run of up to 32 slots; the freed slots below the
  // budget and the kept ones past it are listed in the key array itself: an
  // entry's place is never past the slot it is for, and the runs' keys are read
  // before their entries are written.
  uint32_t holes = 0, movers = 0, eq_before = 0;
  const int run = min(32, (n + kEvThreads - 1) / kEvThreads);
  for (int j0 = 0; j0 < n; j0 += run * kEvThreads) {
    const int j1 = j0 + tid * run;
    uint32_t gt = 0, eq = 0;
    if (run == 32) {
      const uint32_t *p = keys + ev_at(j1);        // (a run does not cross a word of padding)
#pragma unroll
      for (int i = 0; i < 32; i++) {
        const uint32_t k = j1 + i < n ? p[i] : 0;
        gt |= k > prefix ? 1u << i : 0;
        eq |= k == prefix ? 1u << i : 0;
      }
    } else {
      for (int i = 0; i < run && j1 + i < n; i++) {
        const uint32_t k = keys[ev_at(j1 + i)];
        gt |= (uint32_t)(k > prefix) << i;
        eq |= (uint32_t)(k == prefix) << i;
      }
    }
    const int below = min(max(a.budget - j1, 0), 32), inside = min(max(n - j1, 0), run);   // slots of the run
    const uint32_t low = below == 32 ? 0xffffffffu : (1u << below) - 1;
    const uint32_t real = inside == 32 ? 0xffffffffu : (1u << inside) - 1;
    gt &= real;
    eq &= real;
    uint32_t total, keep = gt | eq;
    if (equal != need) {
      uint32_t er = eq_before + scan_excl(__popc(eq), wsum, &total);
      eq_before += total;
      keep = gt;
      for (uint32_t m = eq; m && er < need; m &= m - 1, er++) keep |= m & -m;
    }
    uint32_t hole = ~keep & low & real, mover = keep & ~low & real;
    uint32_t at = scan_excl((uint32_t)__popc(hole) | (uint32_t)__popc(mover) << 16, wsum, &total);
    uint32_t ha = holes + (at & 0xffffu), ma = a.budget + movers + (at >> 16);
    if (a.most) {
      int32_t *to = a.to + (int64_t)blockIdx.x * a.most, *from = a.from + (int64_t)blockIdx.x * a.most - a.budget;
      for (; hole; hole &= hole - 1) to[ha++] = j1 + __ffs(hole) - 1;
      for (; mover; mover &= mover - 1) from[ma++] = j1 + __ffs(mover) - 1;
    } else {
      for (; hole; hole &= hole - 1) keys[ev_at(ha++)] = j1 + __ffs(hole) - 1;
      for (; mover; mover &= mover - 1) keys[ev_at(ma++)] = j1 + __ffs(mover) - 1;
    }
    holes += total & 0xffffu;
    movers += total >> 16;
  }
  __syncthreads();
  if (a.most) {
    if (tid == 0) a.count[blockIdx.x] = holes;
    return;
  }
  // a thread takes one 16-byte piece of k or v, or the four words
  const int per = c.rb / 16, units = 2 * per + 1;
  for (uint32_t i = tid; i < holes * units; i += kEvThreads) {
    const uint32_t m = i / units, u = i - m * units;
    const int64_t dst = lrow + row_of(c, b, h, keys[ev_at(m)]), src = lrow + row_of(c, b, h, keys[ev_at(a.budget + m)]);
    if (u < (uint32_t)(2 * per)) {
      uint8_t *x = u < (uint32_t)per ? c.k : c.v;
      const int q = u < (uint32_t)per ? u : u - per;
      reinterpret_cast<uint4 *>(x + dst * c.rb)[q] = reinterpret_cast<const uint4 *>(x + src * c.rb)[q];
    } else {
      const uint32_t kg = c.kg[src], vg = c.vg[src];
      const float w = c.weight[src];
      const int p = c.pos[src];
      c.kg[dst] = kg;
      c.vg[dst] = vg;
      c.weight[dst] = w;
      c.pos[dst] = p;
    }
  }
}

// The moves, evenly over the GPU (a head's selection leaves it waiting for the
// slowest): a warp takes 32 of a head's, a lane finds one's rows, and the lanes
// then copy the rows' 16-byte pieces side by side.  Sources lie past the budget
// and destinations below it, so loads may pass stores.  Bound by HBM: 512 heads'
// 950,000 rows of head dim 128 cut from 16001 to 2048, 75 us at 5.8 TB/s of DRAM
// traffic, of which 60 % is asked for: a row's four 4-byte fields each pull 64
// bytes.
constexpr int kMvThreads = 256;
__global__ void __launch_bounds__(kMvThreads) kv4_move_kernel(EvArgs a) {
  pdl_trigger();
  const Cache &c = a.c;
  const int chunks = (a.most + kMvThreads - 1) / kMvThreads, lane = threadIdx.x & 31;
  const int64_t head = blockIdx.x / chunks;
  const int m0 = (blockIdx.x - (int)(head * chunks)) * kMvThreads + (threadIdx.x & ~31);
  const int h = (int)(head % c.nKV);
  const int64_t r = head / c.nKV, b = r % a.B, lrow = r / a.B * c.blocks * c.nKV * c.bs;
  pdl_wait();
  const int count = (int)min(a.count[head], (uint32_t)a.most);
  if (m0 >= count) return;
  const bool on = m0 + lane < count;
  int64_t src = 0, dst = 0;
  uint4 w;
  if (on) {
    // (inside the cache whatever another call made of the workspace)
    const uint32_t last = (uint32_t)c.cap - 1;
    src = lrow + max(row_of(c, b, h, min((uint32_t)a.from[head * a.most + m0 + lane], last)), (int64_t)0);
    dst = lrow + max(row_of(c, b, h, min((uint32_t)a.to[head * a.most + m0 + lane], last)), (int64_t)0);
    w = make_uint4(c.kg[src], c.vg[src], __float_as_uint(c.weight[src]), (uint32_t)c.pos[src]);
  }
  const int per = c.rb / 16, pieces = min(32, count - m0) * per;
#pragma unroll
  for (int v = 0; v < 2; v++) {
    uint8_t *codes = v ? c.v : c.k;
    for (int p0 = 0; p0 < pieces; p0 += 32 * kEvPieces) {
      uint4 x[kEvPieces];
      int64_t to[kEvPieces];
#pragma unroll
      for (int i = 0; i < kEvPieces; i++) {
        const int p = p0 + 32 * i + lane, m = p / per, u = p - m * per;
        const int64_t from = __shfl_sync(0xffffffffu, src, m & 31) * c.rb + 16 * u;
        to[i] = __shfl_sync(0xffffffffu, dst, m & 31) * c.rb + 16 * u;
        if (p < pieces) x[i] = *reinterpret_cast<const uint4 *>(codes + from);
      }
#pragma unroll
      for (int i = 0; i < kEvPieces; i++)
        if (p0 + 32 * i + lane < pieces) *reinterpret_cast<uint4 *>(codes + to[i]) = x[i];
    }
  }
  if (on) {
    c.kg[dst] = w.x;
    c.vg[dst] = w.y;
    c.weight[dst] = __uint_as_float(w.z);
    c.pos[dst] = (int)w.w;
  }
}

// Words of workspace: keys that do not fit in shared memory; the lists of moves
// where a head can have more than kEvInline.
struct EvWork {
  int64_t keys, lists;
  int most;
};
EvWork ev_work(const Cache &c, int B, int budget) {
  const int64_t heads = c.layers * B * c.nKV, most = c.cap - budget < budget ? c.cap - budget : budget;
  EvWork w;
  w.keys = c.cap <= kEvSmemSlots ? 0 : heads * ev_at((int)c.cap);
  w.most = most > kEvInline ? (int)most : 0;
  w.lists = w.most ? heads * (2 * w.most + 1) : 0;
  return w;
}

}  // namespace
}  // namespace kv4
}  // namespace fcu

using namespace fcu;
using namespace fcu::kv4;

// f(W) for rows of W 16-byte pieces
#define FCU_KV4_ROWS(f, rb)   \
  switch ((rb) / 16) {        \
    case 1: f(1); break;      \
    case 2: f(2); break;      \
    case 3: f(3); break;      \
    case 4: f(4); break;      \
    case 6: f(6); break;      \
    default: f(8); break;     \
  }

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
  cudaError_t e = cudaSuccess;
#define FCU_CASE(W)                                                                                             \
  e = launch_pdl(a.c.dH == 32 * W ? kv4_put_kernel<W, true> : kv4_put_kernel<W, false>, dim3((unsigned)grid), \
                 dim3(kPutThreads), 0, ctx->stream, a)
  FCU_KV4_ROWS(FCU_CASE, a.c.rb)
#undef FCU_CASE
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
  const int64_t grid = (int64_t)B * ((T + kValTokens - 1) / kValTokens);
  FCU_REQUIRE(grid <= INT_MAX, "fcu_kv4_values: %d x %d tokens in one call", B, T);
  cudaError_t e = cudaSuccess;
#define FCU_CASE(W) e = launch_pdl(kv4_values_kernel<W>, dim3((unsigned)grid), dim3(kValThreads), 0, ctx->stream, a)
  FCU_KV4_ROWS(FCU_CASE, a.c.rb)
#undef FCU_CASE
  FCU_CHECK_CUDA(e);
  note_launch();
  return FCU_OK;
}

int64_t fcu_kv4_evict_work(fcu_ctx *ctx, const fcu_kv4 *cache, int B, int budget) {
  Cache c;
  if (!ctx || B < 0 || budget < 1 || view("fcu_kv4_evict_work", cache, B, false, &c)) return -1;
  const EvWork w = ev_work(c, B, budget);
  return 4 * (w.keys + w.lists);
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
  const EvWork w = ev_work(a.c, B, budget);
  const int64_t need = 4 * (w.keys + w.lists), heads = a.c.layers * B * a.c.nKV;
  FCU_REQUIRE(need == 0 || (work && work_bytes >= need && ((uintptr_t)work & 3) == 0),
              "fcu_kv4_evict: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)need);
  const int64_t moves = heads * ((w.most + kMvThreads - 1) / kMvThreads);
  FCU_REQUIRE(heads <= INT_MAX && moves <= INT_MAX, "fcu_kv4_evict: %lld heads in one call", (long long)heads);
  a.lens = seq_lens;
  a.B = B;
  a.budget = budget;
  a.recent = recent;
  a.new_lens = new_lens;
  a.keys = (uint32_t *)work;
  a.most = w.most;
  if (w.most) {
    a.count = a.keys + w.keys;
    a.to = (int32_t *)(a.count + heads);
    a.from = a.to + heads * w.most;
  }
  const bool vec = a.c.bs % 4 == 0 && (((uintptr_t)a.c.weight | (uintptr_t)a.c.pos) & 15) == 0;
  void (*kernel)(EvArgs);
  if (w.keys) kernel = vec ? kv4_evict_kernel<false, true, 2> : kv4_evict_kernel<false, false, 2>;
  else if (a.c.cap <= 8192) kernel = vec ? kv4_evict_kernel<true, true, 3> : kv4_evict_kernel<true, false, 3>;
  else kernel = vec ? kv4_evict_kernel<true, true, 2> : kv4_evict_kernel<true, false, 2>;
  static bool set[64] = {false};
  if (!set[ctx->device & 63]) {
    const int most = ev_at(kEvSmemSlots) * 4;
    const cudaFuncAttribute smem = cudaFuncAttributeMaxDynamicSharedMemorySize;
    FCU_CHECK_CUDA(cudaFuncSetAttribute(kv4_evict_kernel<true, true, 2>, smem, most));
    FCU_CHECK_CUDA(cudaFuncSetAttribute(kv4_evict_kernel<true, false, 2>, smem, most));
    set[ctx->device & 63] = true;
  }
  const cudaError_t e = launch_pdl(kernel, dim3((unsigned)heads), dim3(kEvThreads),
                                   w.keys ? 0 : (size_t)ev_at((int)a.c.cap) * 4, ctx->stream, a);
  FCU_CHECK_CUDA(e);
  if (moves) {
    note_launch();
    FCU_CHECK_CUDA(launch_pdl(kv4_move_kernel, dim3((unsigned)moves), dim3(kMvThreads), 0, ctx->stream, a));
  }
  note_launch();
  return FCU_OK;
}

}  // extern "C"
