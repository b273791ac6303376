// Beam search on the device: the selection over beams x vocabulary
// (fcu_beam_step) and the reordering of the beams' caches after it
// (fcu_cache_reorder).  The reference samples one sequence on the host
// (src/L8/sampling.js:28-96) and has no beam search.
#include <float.h>

#include "common.cuh"

namespace fcu {
namespace {

// ------------------------------------------------------------------ selection
// Two kernels.  beam_rows reads every logit once: a warp walks 512 logits at a
// time of one slice of one row, with a running maximum and sum of exponentials
// per lane, and lists the tokens whose logits could be among the slice's W best.
// What they have to reach: every lane keeps its largest logit so far, every warp
// the (W / warps)-th largest of those, and W of the slice's logits reach the
// least of the warps' values, about the W-th largest so far; of n logits in no
// particular order some 2 W ln(n / 4096) get past it after the first 4096.  A
// warp's list is cut down to its W best when it is full and at the end.
// beam_merge, one CTA per sequence, turns the slices' sums into each row's
// log-sum-exp and picks the W best of the W rows' W best.  Within a row the
// candidates order as the logits do, so W per slice are enough (a row whose scores
// tie past its W-th best logit is read once more).  The bound is
// reading the logits (HBM): 32 x 8 rows of 100003, 102 MB, take 30 us, 27 of
// them beam_rows (3.8 TB/s, issue slots 58 % busy; 9 us more with sorted lists kept
// in registers, a bound per warp; 4 more with three tiles of a warp in shared memory
// in place of one ahead in registers); 4 rows of 32000 take 9 us, all latency.
constexpr int kBeamThreads = 256;
constexpr int kBeamWarps = kBeamThreads / 32;
constexpr int kMaxW = 32;
constexpr int kTile = 512;                          // logits a warp takes at a time
constexpr int kMaxSlices = 64;
constexpr int kAgain = 32;                          // loads in flight of a lane that reads a tied row again
constexpr int kFound = 64;                          // tokens a warp lists: kMaxW and 32 more at least
constexpr float kLog2e = 1.4426950408889634f;

using Key = unsigned long long;

// Larger logit, larger key; equal logits (0 and -0 too), lower token first.  0
// is below every key.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// (0 gives -inf)
__device__ __forceinline__ float bits_float(uint32_t u) {
  return u == 0 ? -INFINITY : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ Key beam_key(float x, uint32_t token) {
  return (Key)order_bits(x) << 32 | (0xffffffffu - token);
}
__device__ __forceinline__ float key_logit(Key k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

struct BeamArgs {
  const float *logits;
  int64_t ld;
  const float *scores;
  const uint8_t *done;
  int V, B, W, eos, slices;
  int slice;             // logits per slice
  float2 *sums;          // [rows][slices]: M, the maximum, and the sum of exp(x - M)
  Key *best;             // [rows][slices][W]
  float *out_scores;
  int32_t *tokens, *parents;
  uint8_t *out_done;
};

// e^(x - m).  The difference is taken first: x log2 e leaves fp32 for finite x
// (masks of the type's lowest value among them).
__device__ __forceinline__ float beam_exp(float x, float m) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((x - m) * kLog2e));
  return y;
}

// Four logits from p on, those of tokens in [v0, v1) (v: the first one's); the others -inf.
__device__ __forceinline__ float4 load4(const float *p, int v, int v0, int v1) {
  if (v >= v0 && v + 4 <= v1) return __ldcs(reinterpret_cast<const float4 *>(p));
  float4 f = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  if (v >= v0 && v < v1) f.x = p[0];
  if (v + 1 >= v0 && v + 1 < v1) f.y = p[1];
  if (v + 2 >= v0 && v + 2 < v1) f.z = p[2];
  if (v + 3 >= v0 && v + 3 < v1) f.w = p[3];
  return f;
}

// Leaves a warp's n <= kFound tokens of a row the W best in order, their logits
// read again; returns how many.  (Not inlined: a run of tiles rarely needs it.)
__device__ __noinline__ int prune(const float *x, uint32_t *found, Key *keys, int n, int W) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  Key k0 = 0, k1 = 0;
  if (lane < n) k0 = beam_key(x[found[lane]], found[lane]);
  if (lane + 32 < n) k1 = beam_key(x[found[lane + 32]], found[lane + 32]);
  keys[lane] = k0;
  keys[lane + 32] = k1;
  __syncwarp();
  int r0 = 0, r1 = 0;
#pragma unroll 4
  for (int j = 0; j < n; j++) {
    const Key k = keys[j];
    r0 += k > k0;
    r1 += k > k1;
  }
  __syncwarp();
  if (k0 && r0 < W) {
    keys[r0] = k0;
    found[r0] = 0xffffffffu - (uint32_t)k0;
  }
  if (k1 && r1 < W) {
    keys[r1] = k1;
    found[r1] = 0xffffffffu - (uint32_t)k1;
  }
  __syncwarp();
  return n < W ? n : W;
}

__global__ void __launch_bounds__(kBeamThreads, 4) beam_rows_kernel(BeamArgs a) {
  pdl_trigger();
  __shared__ uint32_t found[kBeamWarps][kFound];
  __shared__ Key keys[kBeamWarps][kFound];
  __shared__ float red_m[kBeamWarps], red_s[kBeamWarps];
  // order_bits of what W / (the warps with tiles) of a warp's lanes have met at least
  __shared__ uint32_t reached[kBeamWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.W;
  const int64_t row = blockIdx.y;
  const int v0 = blockIdx.x * a.slice, v1 = (int)min((int64_t)a.V, (int64_t)v0 + a.slice);
  pdl_wait();
  const float *x = a.logits + row * a.ld;
  // tiles start where a 16-byte line does: at most three tokens before v0
  const int skew = (int)(((uintptr_t)(x + v0) >> 2) & 3);
  // This lane's.  M starts at the type's lowest value: terms of -inf are 0 from there
  // on and a NaN is one, wherever it lies, so that no sum has to be left out.
  float M = -FLT_MAX, s = 0.f;
  uint32_t *mine = found[warp];              // tokens
  int n = 0;                                 // in it
  float least = -INFINITY;                   // no smaller logit is among the slice's W best
  int64_t t0 = (int64_t)v0 - skew + warp * kTile;
  float4 next[4];
  auto fetch = [&](int64_t t) {
    if (t >= v0 && t + kTile <= v1) {
      const float4 *p = reinterpret_cast<const float4 *>(x + t) + lane;
#pragma unroll
      for (int i = 0; i < 4; i++) next[i] = __ldcs(p + 32 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int64_t v = t + 128 * i + 4 * lane;
        next[i] = v < v1 ? load4(x + v, (int)v, v0, v1) : float4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      }
    }
  };
  // the nth largest (of different ones) of the lanes' order bits, or 0
  auto nth = [&](uint32_t bits, int n) {
    uint32_t w_th = 0;
    for (int i = 0; i < n && (i == 0 || w_th); i++) {
      w_th = __reduce_max_sync(0xffffffffu, bits);
      if (bits == w_th) bits = 0;
    }
    return w_th;
  };
  fetch(t0);
  if (threadIdx.x < kBeamWarps) reached[threadIdx.x] = 0xffffffffu;
  __syncthreads();
  // W of the slice's logits reach the least of the warps' `reached`.  A warp raises
  // its own with each tile and reads the others' as they stand.
  const int warps = max(1, min(kBeamWarps, (v1 - v0 + skew + kTile - 1) / kTile)), share = (W + warps - 1) / warps;
  float most = -INFINITY;                    // the lane's largest logit
#pragma unroll
  for (int i = 0; i < 4; i++) most = fmaxf(fmaxf(fmaxf(most, next[i].x), fmaxf(next[i].y, next[i].z)), next[i].w);
  if (warp < warps) {
    const uint32_t bits = nth(order_bits(most), share);
    if (lane == 0) reached[warp] = bits;
  }
  __syncthreads();
  for (; t0 < v1; t0 += kTile * kBeamWarps) {
    float f[16];
#pragma unroll
    for (int i = 0; i < 4; i++)
      f[4 * i] = next[i].x, f[4 * i + 1] = next[i].y, f[4 * i + 2] = next[i].z, f[4 * i + 3] = next[i].w;
    fetch(t0 + kTile * kBeamWarps);
    float top = -INFINITY;                   // (fmaxf passes a NaN over)
#pragma unroll
    for (int i = 0; i < 16; i++) top = fmaxf(top, f[i]);
    const float M1 = fmaxf(M, top);
    float ts = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) ts += beam_exp(f[i], M1);
    s = s * beam_exp(M, M1) + ts;
    M = M1;
    most = fmaxf(most, top);
    const uint32_t bits = nth(order_bits(most), share);
    if (lane == 0) *(volatile uint32_t *)&reached[warp] = bits;
    const uint32_t all = *(volatile uint32_t *)&reached[lane % kBeamWarps];
    least = fmaxf(least, bits_float(__reduce_min_sync(0xffffffffu, all)));
    const uint32_t hit = __ballot_sync(0xffffffffu, top >= least);
    if (hit == 0) continue;
    // no logit below the W-th largest of the lanes' maxima is among the W best
    if (__popc(hit) > W) {
      const uint32_t w_th = nth(order_bits(top), W);
      if (w_th) least = fmaxf(least, bits_float(w_th));
    }
    uint32_t is = 0;                         // the lane's logits that reach it
#pragma unroll
    for (int i = 0; i < 16; i++) is |= f[i] >= least ? 1u << i : 0;
    if (t0 < v0 || t0 + kTile > v1)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int64_t v = t0 + 128 * (i / 4) + 4 * lane + i % 4;
        if (v < v0 || v >= v1) is &= ~(1u << i);
      }
    float own = -INFINITY;                   // the W-th best of a warp that has W
    bool full = false;
    while (true) {
      const uint32_t who = __ballot_sync(0xffffffffu, is);
      if (who == 0) break;
      if (n + __popc(who) > kFound) {
        n = prune(x, mine, keys[warp], n, W);
        full = true;
        own = key_logit(keys[warp][W - 1]);
        least = fmaxf(least, own);
      }
      if (is) {
        const int i = __ffs(is) - 1;
        mine[n + __popc(who & ((1u << lane) - 1))] = (uint32_t)t0 + 128 * (i / 4) + 4 * lane + i % 4;
        is &= is - 1;
      }
      n += __popc(who);
    }
    // later tiles hold higher tokens: of theirs, only logits above this warp's own
    // W-th are wanted (another's may be of later tokens)
    if (full && own >= least) least = bits_float(order_bits(own) + 1);
  }
  n = prune(x, mine, keys[warp], n, W);
  // the slice's maximum and sum: lanes, then warps, in a fixed order
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float oM = __shfl_xor_sync(0xffffffffu, M, o), os = __shfl_xor_sync(0xffffffffu, s, o);
    const float M1 = fmaxf(M, oM);
    s = s * beam_exp(M, M1) + os * beam_exp(oM, M1);
    M = M1;
  }
  if (lane == 0) red_m[warp] = M, red_s[warp] = s;
  __syncthreads();
  const int64_t at = row * a.slices + blockIdx.x;
  if (threadIdx.x == 0) {
    float M1 = red_m[0], S = 0.f;
    for (int w = 1; w < kBeamWarps; w++) M1 = fmaxf(M1, red_m[w]);
    for (int w = 0; w < kBeamWarps; w++) S += red_s[w] * beam_exp(red_m[w], M1);
    a.sums[at] = make_float2(M1, S);
  }
  // the warps' lists are sorted and share no key: one's rank is its own place
  // plus what every other list has above it
  if (threadIdx.x < W) a.best[at * W + threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < kBeamWarps * W; i += kBeamThreads) {
    const Key k = keys[i / W][i % W];
    int rank = i % W;
    for (int w = 0; w < kBeamWarps && rank < W; w++)
      if (w != i / W)
        for (int j = 0; j < W && keys[w][j] > k; j++) rank++;
    if (k && rank < W) a.best[at * W + rank] = k;
  }
}

__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(BeamArgs a) {
  pdl_trigger();
  extern __shared__ __align__(16) Key raw[];           // [W][slices][W]
  __shared__ Key best[kMaxW][kMaxW];
  __shared__ double score[kMaxW][kMaxW];
  __shared__ int token[kMaxW][kMaxW];                  // -1: no candidate
  __shared__ uint8_t order[kMaxW][kMaxW];              // a row's candidates, best first
  __shared__ float top_s[kMaxW];                       // a row's largest logit
  __shared__ double log_s[kMaxW];                      // and the log of its sum of exp(x - the largest)
  __shared__ bool tied[kMaxW];                         // a logit below the W-th best scores what that one does
  __shared__ int again[kBeamWarps][kMaxW], agains[kBeamWarps];
  const int tid = threadIdx.x, lane = tid & 31, W = a.W, per = a.slices * W, N = W * per;
  const int64_t b = blockIdx.x;
  for (int i = tid; i < W * W; i += kBeamThreads) best[i / W][i % W] = 0;
  pdl_wait();
  for (int i = tid; i < N; i += kBeamThreads) raw[i] = a.best[b * N + i];
  for (int w = tid >> 5; w < W; w += kBeamWarps) {
    float M = -FLT_MAX, S = 0.f;
    for (int i = lane; i < a.slices; i += 32) {
      const float2 x = a.sums[(b * W + w) * a.slices + i];
      const float M1 = fmaxf(M, x.x);
      S = S * beam_exp(M, M1) + x.y * beam_exp(x.x, M1);
      M = M1;
    }
    const float top = warp_max(M);
    S = warp_sum(S * beam_exp(M, top));
    // (not finite where a logit was NaN or +inf, or all were -inf)
    if (lane == 0) top_s[w] = top, log_s[w] = log((double)S);
  }
  __syncthreads();
  // A row's W best of its slices' sorted lists.  Few lists: a key's rank is its
  // own place plus what every other list has above it.  Many: W times the largest
  // of their heads, of which a lane has up to two.  (Whole steps by rank and by heads:
  // 2 lists of 8 29.7 and 31.7 us, 2 of 32 71.0 and 86.9; 5 of 8 14.8 and 12.5, 8 of 32
  // 168 and 45.8, 16 of 4 10.9 and 8.8.)
  if (a.slices <= 2) {
    for (int i = tid; i < N; i += kBeamThreads) {
      const int w = i / per, mine = (i - w * per) / W;
      const Key k = raw[i];
      int rank = i % W;
      for (int x = 0; x < a.slices && rank < W; x++)
        if (x != mine)
          for (int j = 0; j < W && raw[w * per + x * W + j] > k; j++) rank++;
      if (k && rank < W) best[w][rank] = k;
    }
  } else {
    for (int w = tid >> 5; w < W; w += kBeamWarps) {
      const Key *row = raw + w * per;
      int at0 = 0, at1 = 0;
      Key h0 = lane < a.slices ? row[lane * W] : 0, h1 = lane + 32 < a.slices ? row[(lane + 32) * W] : 0;
      for (int r = 0; r < W; r++) {
        const Key mine = h0 > h1 ? h0 : h1;
        const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32));
        const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32) == hi ? (uint32_t)mine : 0);
        const Key top = (Key)hi << 32 | lo;
        if (top == 0) break;
        if (lane == 0) best[w][r] = top;
        if (h0 == top) h0 = ++at0 < W ? row[lane * W + at0] : 0;
        else if (h1 == top) h1 = ++at1 < W ? row[(lane + 32) * W + at1] : 0;
      }
    }
  }
  __syncthreads();
  auto value = [&](int w, double cum, float logit) { return cum + (((double)logit - top_s[w]) - log_s[w]) + 0.0; };
  for (int i = tid; i < W * W; i += kBeamThreads) {
    const int w = i / W, r = i - w * W;
    const double cum = a.scores[b * W + w];
    bool more = false;
    const bool done = a.done[b * W + w] != 0;
    // a beam with nothing finite to offer stands for its lowest tokens
    const bool dead = !isfinite(cum) || (!done && !isfinite(log_s[w]));
    double v = -INFINITY;
    int tok = r < a.V ? r : -1;
    if (done && !dead) {
      // eos, then the other tokens in order
      tok = r >= a.V ? -1 : r == 0 ? a.eos : r - (r <= a.eos);
      if (r == 0) v = cum;
    } else if (!dead) {
      const Key k = best[w][r];
      tok = k ? (int)(0xffffffffu - (uint32_t)k) : -1;
      v = value(w, cum, key_logit(k));
      if (!isfinite(v)) v = -INFINITY;
      const uint32_t u = (uint32_t)(k >> 32), below = u == order_bits(0.f) ? u - 2 : u - 1;   // (u - 1 there: -0)
      more = r == W - 1 && k && v > -INFINITY && value(w, cum, bits_float(below)) == v;
    }
    score[w][r] = v + 0.0;
    token[w][r] = tok;
    if (r == W - 1) tied[w] = more;
  }
  __syncthreads();
  // Where the beam's score or its log-sum-exp swallows the difference of two logits
  // (a score of -1e30, logits of 1e-20), tokens that the row's W best logits do not
  // hold may tie with the last of those: the lowest of all that score as it does
  // take its place and those of its equals in the list, if any of those are chosen.  A
  // warp looks through an eighth of the row.  (One beam over logits less their maximum,
  // whose best is 0, is such a row: 32 x 1 x 100003 42 us, 11 without, 196 with one warp
  // to a row; 1 x 1 x 32000 13.7, 6.9 and 30.7.)
  for (uint32_t m = __ballot_sync(0xffffffffu, lane < W && tied[lane]); m; m &= m - 1) {
    const int w = __ffs(m) - 1;
    const double last = score[w][W - 1];
    int above = 0;                                     // candidates before the first of them
    for (int i0 = 0; i0 < W * W; i0 += kBeamThreads) {
      const int i = i0 + tid, x = i / W;
      above += __syncthreads_count(i < W * W && token[x][i % W] >= 0 &&
                                   (score[x][i % W] > last || (score[x][i % W] == last && x < w)));
    }
    if (above >= W) continue;                          // none of them is chosen
    const float *x = a.logits + (b * W + w) * a.ld;
    const double cum = a.scores[b * W + w];
    const int first = __popc(__ballot_sync(0xffffffffu, lane < W && score[w][lane < W ? lane : 0] > last));
    // no logit below `low` scores `last`: value() rounds by far less than 2^-50 of its terms
    const float best_w = key_logit(best[w][W - 1]);
    const double off = 0x1p-50 * (fabs(cum) + fabs((double)top_s[w]) + fabs((double)best_w) + fabs(log_s[w]));
    const float low = __double2float_rd((double)best_w - off);
    const int part = (a.V + kBeamWarps - 1) / kBeamWarps, v0 = (tid >> 5) * part, v1 = min(a.V, v0 + part);
    int n = 0;
    for (int t0 = v0; t0 < v1 && n < W - first; t0 += 32 * kAgain) {
      float f[kAgain];
#pragma unroll
      for (int i = 0; i < kAgain; i++) {
        const int t = t0 + 32 * i + lane;
        f[i] = t < v1 ? x[t] : -INFINITY;
      }
      bool any = false;
#pragma unroll
      for (int i = 0; i < kAgain; i++) any |= f[i] >= low;
      if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
      for (int i = 0; i < kAgain; i++) {
        const bool hit = f[i] >= low && value(w, cum, f[i]) == last;
        const uint32_t who = __ballot_sync(0xffffffffu, hit);
        const int place = n + __popc(who & ((1u << lane) - 1));
        if (hit && place < W - first) again[tid >> 5][place] = t0 + 32 * i + lane;
        n += __popc(who);
      }
    }
    if (lane == 0) agains[tid >> 5] = min(n, W - first);
    __syncthreads();
    int at = first;
    for (int i = 0; i < (tid >> 5); i++) at += agains[i];
    if (lane < agains[tid >> 5] && at + lane < W) token[w][at + lane] = again[tid >> 5][lane];
    __syncthreads();
  }
  // A row's scores fall as its logits do, but where the beam's score swallows the
  // difference of two logits they tie, and the lower token is first.  (Those of
  // -inf are in order: equal logits or none.)
  for (int i = tid; i < W * W; i += kBeamThreads) {
    const int w = i / W, r = i - w * W;
    const double v = score[w][r];
    int rank = r;
    if (v > -INFINITY && ((r > 0 && score[w][r - 1] == v) || (r + 1 < W && score[w][r + 1] == v))) {
      rank = 0;
      for (int j = 0; j < W && token[w][j] >= 0; j++)
        rank += score[w][j] > v || (score[w][j] == v && token[w][j] < token[w][r]);
    }
    order[w][rank] = (uint8_t)r;
  }
  __syncthreads();
  // W times the best of the rows' heads, a lane's row each; ties to the lowest row
  if (tid >= 32) return;
  auto bits = [&](int at) -> Key {             // orders as the score; 0: the row has no more
    const int r = at < W ? order[lane][at] : 0;
    if (at >= W || token[lane][r] < 0) return 0;
    const Key u = __double_as_longlong(score[lane][r]);
    return u >> 63 ? ~u : u | (Key)1 << 63;
  };
  int at = 0;
  Key head = lane < W ? bits(0) : 0;
  for (int i = 0; i < W; i++) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 32) == hi ? (uint32_t)head : 0);
    const uint32_t who = __ballot_sync(0xffffffffu, head == ((Key)hi << 32 | lo));
    if (lane == __ffs(who) - 1 && head != 0) {
      const int r = order[lane][at];
      const int64_t o = b * W + i;
      a.out_scores[o] = (float)score[lane][r];
      a.tokens[o] = token[lane][r];
      a.parents[o] = lane;
      a.out_done[o] = a.done[b * W + lane] != 0 || token[lane][r] == a.eos;
      head = bits(++at);
    }
  }
}

// Slices per row: enough warps for about 24 on each SM; of more than 1024 logits each
// (about 2048 in long rows), so that three or four of a CTA's eight warps have a tile at
// least; and few enough that the merge ranks at most 256 survivors a row.
int beam_slices(int num_sms, int B, int W, int64_t V) {
  const int64_t rows = (int64_t)B * W > 0 ? (int64_t)B * W : 1;
  int64_t s = ((int64_t)num_sms * 24 / kBeamWarps + rows - 1) / rows;
  const int64_t most = (V + kTile * kBeamWarps / 2 - 1) / (kTile * kBeamWarps / 2);
  s = s < most ? s : most;
  s = s < 256 / W ? s : 256 / W;
  return (int)(s < 1 ? 1 : s > kMaxSlices ? kMaxSlices : s);
}

// ------------------------------------------------------------------ reordering
// A warp takes up to 512 D bytes of one head of one block at a time, at the same
// place of all beams of a sequence: it reads them from the beams that another
// beam continues into its part of shared memory, all copies in flight at once,
// then writes the beams that continue another.  A lane writes only places it has
// read itself and no other warp touches them, so the permutation (with
// repetitions) is done in place without a barrier.  The bound is HBM: every
// beam that is continued is read once, every beam that changes written once.
// 12 layers, 16 x 4 beams of 1003 slots, 4 heads of 64: 62 us (4.8 TB/s).
constexpr int kReThreads = 128;
constexpr int kReWarps = kReThreads / 32;

struct ReArgs {
  uint8_t *base[8];
  int64_t heads[8], unit[8];
  int n_arrays;
  int64_t layers, blocks;
  const int32_t *table, *parents, *lens;
  int bs, mb, B, W;
  int64_t cap;
};

// n <= 16 bytes, a multiple of 4; `wide`: 16-byte aligned
__device__ __forceinline__ void re_load(uint32_t dst, const uint8_t *src, int n, bool wide) {
  if (wide && n == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src));
  } else {
    for (int i = 0; i < n; i += 4)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + i), "l"(src + i));
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

// D: 16-byte pieces of a lane from one beam in one step.
template <int D>
__global__ void __launch_bounds__(kReThreads) cache_reorder_kernel(ReArgs a) {
  pdl_trigger();
  extern __shared__ __align__(16) uint4 hold[];     // [warp][W][D][32]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = a.W;
  const int b = blockIdx.y;
  const int64_t layer = blockIdx.z;
  uint4 *mine = hold + warp * W * D * 32 + lane;
  const uint32_t mine_s = (uint32_t)__cvta_generic_to_shared(mine);
  pdl_wait();
  // lane w: the beam that beam w becomes (itself if it stays) and beam w's length
  int src = lane, len = 0;
  if (lane < W) {
    const int p = a.parents[(int64_t)b * W + lane];
    src = p >= 0 && p < W ? p : lane;
    const int64_t n = a.lens[(int64_t)b * W + lane];
    len = (int)(n < 0 ? 0 : n > a.cap ? a.cap : n);
  }
  const uint32_t moves = __ballot_sync(0xffffffffu, lane < W && src != lane);
  uint32_t needed = 0;
  for (uint32_t m = moves; m; m &= m - 1) needed |= 1u << __shfl_sync(0xffffffffu, src, __ffs(m) - 1);
  if (!needed) return;
  const int longest = __reduce_max_sync(0xffffffffu, needed >> lane & 1 ? len : 0);
  constexpr int chunk = 512 * D;                            // bytes of one step
  for (int x = 0; x < a.n_arrays; x++) {
    const int64_t unit = a.unit[x], seg = a.bs * unit;      // bytes of one head of one block
    const bool wide = seg % 16 == 0;
    const int64_t used = min(seg, longest * unit);          // no block holds more
    const int steps = (int)((used + chunk - 1) / chunk), blks = (longest + a.bs - 1) / a.bs;
    const int64_t items = (int64_t)a.heads[x] * blks * steps;
    for (int64_t i = (int64_t)blockIdx.x * kReWarps + warp; i < items; i += (int64_t)gridDim.x * kReWarps) {
      const int64_t hb = i / steps;
      const int h = (int)(hb / blks), blk = (int)(hb - (int64_t)h * blks);
      const int64_t off = (i - hb * steps) * chunk;
      // lane w: beam w's place of this step and the bytes of it that its length covers
      int64_t at = -1, valid = 0;
      if (lane < W) {
        const int64_t r = (int64_t)b * W + lane;
        int64_t p = r * a.mb + blk;
        if (a.table) {
          p = a.table[p];
          if (p >= a.blocks) p = -1;
        }
        if (p >= 0) at = ((layer * a.blocks + p) * a.heads[x] + h) * seg + off;
        valid = min(seg, ((int64_t)len - (int64_t)blk * a.bs) * unit) - off;
      }
      const int bytes = (int)max((int64_t)0, min((int64_t)chunk, valid));
      for (uint32_t m = needed; m; m &= m - 1) {
        const int w = __ffs(m) - 1;
        const int64_t from = __shfl_sync(0xffffffffu, at, w);
        const int n = __shfl_sync(0xffffffffu, bytes, w);
        if (from < 0) continue;
        const uint8_t *p = a.base[x] + from + 16 * lane;
        const uint32_t to = mine_s + w * D * 512;
        if (wide && n == chunk) {
#pragma unroll
          for (int d = 0; d < D; d++) re_load(to + 512 * d, p + 512 * d, 16, true);
        } else {
          for (int d = 0; d < D && 512 * d + 16 * lane < n; d++)
            re_load(to + 512 * d, p + 512 * d, min(16, n - 512 * d - 16 * lane), wide);
        }
      }
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
      for (uint32_t m = moves; m; m &= m - 1) {
        const int w = __ffs(m) - 1, s = __shfl_sync(0xffffffffu, src, w);
        const int64_t to = __shfl_sync(0xffffffffu, at, w), from = __shfl_sync(0xffffffffu, at, s);
        const int n = __shfl_sync(0xffffffffu, bytes, s);
        if (to < 0 || from < 0) continue;
        uint8_t *p = a.base[x] + to + 16 * lane;
        const uint4 *y = mine + s * D * 32;
        if (wide && n == chunk) {
#pragma unroll
          for (int d = 0; d < D; d++) re_store(p + 512 * d, y + 32 * d, 16, true);
        } else {
          for (int d = 0; d < D && 512 * d + 16 * lane < n; d++)
            re_store(p + 512 * d, y + 32 * d, min(16, n - 512 * d - 16 * lane), wide);
        }
      }
      asm volatile("" ::: "memory");      // `mine` is read before the next step's copies into it
    }
  }
}

}  // namespace
}  // namespace fcu

using namespace fcu;

extern "C" {

int64_t fcu_beam_work(fcu_ctx *ctx, int B, int W, int64_t V) {
  if (!ctx || B < 0 || W < 1 || W > kMaxW || V < 1) return -1;
  const int64_t parts = (int64_t)B * W * beam_slices(ctx->num_sms, B, W, V);
  return parts * (sizeof(float2) + W * sizeof(Key));
}

int fcu_beam_step(fcu_ctx *ctx, const float *logits, int64_t ld, const float *scores, const uint8_t *done, int B,
                  int W, int64_t V, int eos, float *out_scores, int32_t *tokens, int32_t *parents,
                  uint8_t *out_done, void *work, int64_t work_bytes) {
  FCU_CTX(ctx);
  FCU_REQUIRE(B >= 0 && W >= 1 && W <= kMaxW, "fcu_beam_step: %d sequences of %d beams (1..%d)", B, W, kMaxW);
  FCU_REQUIRE(V >= 1 && V <= 1 << 30, "fcu_beam_step: a vocabulary of %lld", (long long)V);
  FCU_REQUIRE(eos >= 0 && eos < V, "fcu_beam_step: eos %d outside the vocabulary", eos);
  FCU_REQUIRE(ld >= V, "fcu_beam_step: row stride %lld too small", (long long)ld);
  FCU_REQUIRE((int64_t)B * W <= 65535, "fcu_beam_step: %d x %d rows in one call", B, W);
  if (B == 0) return FCU_OK;
  FCU_REQUIRE(logits && scores && done && out_scores && tokens && parents && out_done, "fcu_beam_step: null pointer");
  const int64_t R = (int64_t)B * W;
  auto apart = [&](const void *p, int64_t n, const void *q, int64_t m) {
    return (uintptr_t)p + n <= (uintptr_t)q || (uintptr_t)q + m <= (uintptr_t)p;
  };
  const void *outs[4] = {out_scores, tokens, parents, out_done};
  for (int i = 0; i < 4; i++) {
    const int64_t n = i < 3 ? 4 * R : R;
    bool ok = apart(outs[i], n, scores, 4 * R) && apart(outs[i], n, done, R) &&
              apart(outs[i], n, logits, 4 * ((R - 1) * ld + V));
    for (int j = 0; j < i; j++) ok &= apart(outs[i], n, outs[j], 4 * R);
    FCU_REQUIRE(ok, "fcu_beam_step: an output overlaps another or an input");
  }
  const int64_t need = fcu_beam_work(ctx, B, W, V);
  FCU_REQUIRE(work && work_bytes >= need && ((uintptr_t)work & 15) == 0,
              "fcu_beam_step: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)need);
  BeamArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.scores = scores;
  a.done = done;
  a.V = (int)V;
  a.B = B;
  a.W = W;
  a.eos = eos;
  a.slices = beam_slices(ctx->num_sms, B, W, V);
  a.slice = (int)((V + a.slices - 1) / a.slices);
  a.best = (Key *)work;
  a.sums = (float2 *)(a.best + (int64_t)B * W * a.slices * W);
  a.out_scores = out_scores;
  a.tokens = tokens;
  a.parents = parents;
  a.out_done = out_done;
  const size_t smem = (size_t)W * W * a.slices * sizeof(Key);
  static bool set[64] = {false};
  if (!set[ctx->device & 63]) {
    FCU_CHECK_CUDA(cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024));
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
  // 8 KB of shared memory a warp up to 16 beams, 16 KB for 32
  const int depth = W <= 4 ? 4 : W <= 8 ? 2 : 1;
  int64_t most = 0;
  for (int i = 0; i < n_arrays; i++) {
    FCU_REQUIRE(arrays[i].base && ((uintptr_t)arrays[i].base & 15) == 0,
                "fcu_cache_reorder: array %d is null or not 16-byte aligned", i);
    FCU_REQUIRE(arrays[i].heads > 0 && arrays[i].heads <= 65535 && arrays[i].unit > 0 && arrays[i].unit % 4 == 0 &&
                    arrays[i].unit <= 1 << 24 && (int64_t)block_size * arrays[i].unit <= (int64_t)1 << 34,
                "fcu_cache_reorder: array %d of %lld heads, %lld bytes a slot", i, (long long)arrays[i].heads,
                (long long)arrays[i].unit);
    a.base[i] = (uint8_t *)arrays[i].base;
    a.heads[i] = arrays[i].heads;
    a.unit[i] = arrays[i].unit;
    // (sizes in double: their products may pass 64 bits)
    const double bytes = (double)layers * blocks * block_size;
    for (int j = 0; j < i; j++) {
      const uintptr_t p = (uintptr_t)a.base[i], q = (uintptr_t)a.base[j];
      const double first = p < q ? bytes * a.heads[i] * a.unit[i] : bytes * a.heads[j] * a.unit[j];
      FCU_REQUIRE((double)(p < q ? q - p : p - q) >= first,
                  "fcu_cache_reorder: arrays %d and %d overlap", j, i);
    }
    const int64_t chunk = 512 * depth, steps = ((int64_t)block_size * arrays[i].unit + chunk - 1) / chunk;
    const int64_t items = arrays[i].heads * max_blocks * steps;
    most = items > most ? items : most;
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
  // CTAs over a (sequence, layer): about eight waves of them in all, a warp then walks the rest
  const int64_t pairs = (int64_t)B * layers, fill = (8 * 6 * (int64_t)ctx->num_sms + pairs - 1) / pairs;
  int64_t gx = (most + kReWarps - 1) / kReWarps;
  gx = gx < fill ? gx : fill;
  const size_t smem = (size_t)W * depth * kReThreads * 16;
  static bool set[64] = {false};
  if (!set[ctx->device & 63]) {
    FCU_CHECK_CUDA(cudaFuncSetAttribute(cache_reorder_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        kMaxW * kReThreads * 16));
    set[ctx->device & 63] = true;
  }
  void (*kernel)(ReArgs) = cache_reorder_kernel<1>;
  if (depth > 1) kernel = depth == 4 ? cache_reorder_kernel<4> : cache_reorder_kernel<2>;
  FCU_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)gx, B, (unsigned)layers), dim3(kReThreads), smem,
                            ctx->stream, a));
  note_launch();
  return FCU_OK;
}

}  // extern "C"
