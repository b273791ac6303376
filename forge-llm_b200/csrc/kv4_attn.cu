// Attention of one new token per sequence over the 4-bit KV cache
// (fcu_kv4_attn; layout in kv4.cuh).
//
//   s_j = scale (step_j q.c_j + base_j sum q),  p = softmax(s)
//   o_e = sum_j p_j step_j c_je + sum_j p_j base_j
//
// One pass over the cache with a running maximum and sum.  The bound is
// reading the cache: a slot of one kv head is 2 (dH / 2 + 4) bytes, and every
// q head of the group uses it while it is on the chip.
//
// Both products run on mma.sync m16n8k16 with fp16 operands and fp32 sums.
// The codes are exact in fp16 without a conversion: a nibble in the low byte
// of a 16-bit half IS the subnormal c 2^-24 (or 16 c 2^-24), so two ANDs on a
// word give four operands.  The other operand carries 22 bits, x = hi + lo, in
// rows r and r + 8 of the same instruction (heads 0..7 and their remainders),
// whose sums are added in fp32; a power of two keeps it in fp16's range.  (An
// M = 128 tcgen05 tile would want the codes expanded to 16 bits in shared
// memory first, four times the traffic of the codes themselves; from registers
// the legacy pipe is fast enough, one m16n8k16 per 36 bytes of cache.)
//
// Work is cut by tiles of slots, not by sequence: the tiles of all (sequence,
// kv head) segments in a row are dealt in equal runs to as many CTAs as the GPU
// holds, so a ragged batch or one long sequence fill it alike.  A segment that
// lies inside one run is finished there; one cut by run borders leaves pieces
// (o, m, l) that a second kernel merges.
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace fcu {
namespace kv4 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kStages = 2;
constexpr int kHeads = 8;              // q heads of one CTA (rows of the mma tile, twice)
constexpr float kLog2e = 1.4426950408889634f;

// W: a row is W 16-byte units (dP = 32 W elements).
template <int W>
struct Cfg {
  static constexpr int kTile = W <= 4 ? 64 : 32;                  // slots of one warp's step
  static constexpr int kRow = 16 * W;
  static constexpr int kGridStride = kTile / 4 + 4;               // words; slots 4i + t of column t
  static constexpr int kCodes = kTile * kRow;
  static constexpr int kStage = 2 * kCodes + 2 * 16 * kGridStride;
  static constexpr int kCtas = W <= 2 ? 4 : W <= 4 ? 3 : 2;       // per SM, by registers
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kMerge = kWarps * kHeads * (32 * W + 2) * 4;   // the warps' o, m, l at a segment's end
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

struct AttnArgs {
  const float *q;
  int64_t ld_q;
  Cache c;
  const int32_t *lens;
  int B, nH, g;          // g: q heads per kv head
  int gs, hg;            // q heads of one segment, segments per kv head
  int ctas;              // runs (CTAs of the main kernel)
  float scale;
  float *out;
  float *part;           // [ctas][2][kHeads][dH + 2]: o, then m (log2 units) and l
  float2 *ml;            // [B, nH] final m and l, where weights are kept
  float *scores;         // [B, nH, cap] in log2 units, where weights are kept
};

__device__ __forceinline__ int64_t length(const AttnArgs &a, int64_t b) {
  const int64_t n = a.lens[b];
  return n < 0 ? 0 : n > a.c.cap ? a.c.cap : n;
}

// The cut into runs, the same in every kernel of a call: `total` tiles, `per`
// of them to a run.  A run is at least a tile for every warp of the CTA, unless
// no segment is that long.
struct Plan {
  int64_t total, per;
};

// Block-wide; sh: 2 * kWarps int64.
template <int TILE>
__device__ Plan make_plan(const AttnArgs &a, int64_t *sh) {
  const int segs = a.c.nKV * a.hg;
  int64_t total = 0, longest = 0;
  for (int64_t b = threadIdx.x; b < a.B; b += kThreads) {
    const int64_t t = (length(a, b) + TILE - 1) / TILE;
    total += t;
    longest = max(longest, t);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
  }
  if ((threadIdx.x & 31) == 0) {
    sh[threadIdx.x >> 5] = total;
    sh[kWarps + (threadIdx.x >> 5)] = longest;
  }
  __syncthreads();
  total = longest = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    total += sh[w];
    longest = max(longest, sh[kWarps + w]);
  }
  __syncthreads();
  Plan p;
  p.total = total * segs;
  p.per = max((p.total + a.ctas - 1) / a.ctas, min((int64_t)kWarps, longest));
  return p;
}

// A tile's place: sequence, segment of the sequence, tile of the segment.
struct Place {
  int64_t b;
  int seg;
  int64_t tile, tiles;
};

// The place of tile u < total (b = -1 if the lengths have changed since the
// total was taken).  Block-wide, the same for all threads; sh: kThreads int64.
template <int TILE>
__device__ Place find(const AttnArgs &a, int64_t u, int64_t *sh) {
  const int segs = a.c.nKV * a.hg, tid = threadIdx.x;
  int64_t before = 0;
  for (int64_t b0 = 0; b0 < a.B; b0 += kThreads) {
    const int64_t t = b0 + tid < a.B ? (length(a, b0 + tid) + TILE - 1) / TILE : 0;
    int64_t x = t * segs;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if ((tid & 31) >= o) x += y;
    }
    sh[tid] = x;
    __syncthreads();
    for (int w = 0; w < (tid >> 5); w++) x += sh[32 * w + 31];
    __syncthreads();
    sh[tid] = before + x;      // tiles up to and with sequence b0 + tid
    const int hit = __syncthreads_count(before + x <= u);
    if (hit < kThreads) {
      const int64_t first = hit ? sh[hit - 1] : before;
      Place p;
      p.b = b0 + hit;
      p.tiles = (sh[hit] - first) / segs;
      __syncthreads();
      p.seg = (int)((u - first) / p.tiles);
      p.tile = (u - first) - p.seg * p.tiles;
      return p;
    }
    before = sh[kThreads - 1];
    __syncthreads();
  }
  return Place{-1, 0, 0, 0};
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (x, y) as fp16 pairs, hi and the remainders
__device__ __forceinline__ void split(float x, float y, uint32_t *hi, uint32_t *lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  *hi = *reinterpret_cast<const uint32_t *>(&h);
  *lo = *reinterpret_cast<const uint32_t *>(&l);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0));
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0));
}

// Starts the copies of one tile (slots j0 .. j0 + cnt of head h of sequence b)
// into a warp's stage.  Slots past cnt are zero; those of a bad block have NaN
// grids.
template <int W>
__device__ __forceinline__ void issue(const Cache &c, int64_t b, int h, int64_t j0, int cnt, uint8_t *stage) {
  using C = Cfg<W>;
  const int lane = threadIdx.x & 31;
  const uint32_t k_s = (uint32_t)__cvta_generic_to_shared(stage), v_s = k_s + C::kCodes;
  const uint32_t kg_s = v_s + C::kCodes, vg_s = kg_s + 16 * C::kGridStride;
  const int64_t blk = c.mb == 1 ? 0 : (int64_t)((uint32_t)j0 / (uint32_t)c.bs);
  const int off = (int)(j0 - blk * c.bs);
  if (off + cnt <= c.bs) {
    // one block: the tile's rows are contiguous
    const int64_t p = block_of(c, b, blk);
    const bool ok = p >= 0;
    const int64_t row = ok ? (p * c.nKV + h) * c.bs + off : 0;
    const uint8_t *ks = c.k + row * C::kRow, *vs = c.v + row * C::kRow;
#pragma unroll
    for (int i = 0; i < C::kTile * W / 32; i++) {
      const int x = i * 32 + lane;
      const bool on = ok && x / W < cnt;
      cp_async16(k_s + 16 * x, on ? ks + 16 * x : c.k, on);
      cp_async16(v_s + 16 * x, on ? vs + 16 * x : c.v, on);
    }
#pragma unroll
    for (int i = 0; i < C::kTile / 32; i++) {
      const int x = i * 32 + lane;
      const uint32_t at = 4 * ((x & 3) * C::kGridStride + (x >> 2));
      const bool on = ok && x < cnt;
      if (ok || x >= cnt) {
        cp_async4(kg_s + at, on ? c.kg + row + x : c.kg, on);
        cp_async4(vg_s + at, on ? c.vg + row + x : c.vg, on);
      } else {
        *reinterpret_cast<uint32_t *>(stage + 2 * C::kCodes + at) = kNanGrid;
        *reinterpret_cast<uint32_t *>(stage + 2 * C::kCodes + 16 * C::kGridStride + at) = kNanGrid;
      }
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < C::kTile * W / 32; i++) {
      const int x = i * 32 + lane, j = x / W;
      const int64_t row = j < cnt ? row_of(c, b, h, j0 + j) : -1;
      const int64_t at = row * C::kRow + 16 * (x - j * W);
      cp_async16(k_s + 16 * x, row >= 0 ? c.k + at : c.k, row >= 0);
      cp_async16(v_s + 16 * x, row >= 0 ? c.v + at : c.v, row >= 0);
    }
#pragma unroll 1
    for (int x = lane; x < C::kTile; x += 32) {
      const uint32_t at = 4 * ((x & 3) * C::kGridStride + (x >> 2));
      const int64_t row = x < cnt ? row_of(c, b, h, j0 + x) : -1;
      if (row >= 0 || x >= cnt) {
        cp_async4(kg_s + at, row >= 0 ? c.kg + row : c.kg, row >= 0);
        cp_async4(vg_s + at, row >= 0 ? c.vg + row : c.vg, row >= 0);
      } else {
        *reinterpret_cast<uint32_t *>(stage + 2 * C::kCodes + at) = kNanGrid;
        *reinterpret_cast<uint32_t *>(stage + 2 * C::kCodes + 16 * C::kGridStride + at) = kNanGrid;
      }
    }
  }
}

// N words from shared memory at an address aligned to 4 N bytes' largest power of two
template <int N>
__device__ __forceinline__ void lds(const uint8_t *p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4 *>(p + 4 * i);
      w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint2 x = *reinterpret_cast<const uint2 *>(p + 4 * i);
      w[i] = x.x, w[i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = *reinterpret_cast<const uint32_t *>(p + 4 * i);
  }
}

// In the mma tiles, thread (r = lane / 4, t = lane % 4) of a warp holds head r
// and, of the 8 slots of an n-tile, columns 2t and 2t + 1, which stand for
// slots t and t + 4: then the four t of a V load read four neighbouring rows.
template <int W>
__global__ void __launch_bounds__(kThreads, Cfg<W>::kCtas) kv4_attn_kernel(AttnArgs a) {
  using C = Cfg<W>;
  constexpr int TP = C::kTile, NT = TP / 8, KS = TP / 16, dP = 32 * W;
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ int64_t sh[kThreads];
  const Cache &c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
  uint8_t *ring = sm + warp * kStages * C::kStage;
  pdl_wait();
  for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x)
    if (length(a, b) == 0)
      for (int i = threadIdx.x; i < a.nH * c.dH; i += kThreads) a.out[b * a.nH * c.dH + i] = 0.f;
  const Plan plan = make_plan<TP>(a, sh);
  int64_t u = blockIdx.x * plan.per;
  const int64_t end = min(u + plan.per, plan.total);
  if (u >= end) return;
  Place at = find<TP>(a, u, sh);
  while (at.b >= 0 && at.b < a.B) {
    // this run's part [t0, t1) of the segment
    const int64_t t0 = at.tile, t1 = min(at.tiles, t0 + (end - u));
    const int h = at.seg / a.hg, h0 = h * a.g + (at.seg % a.hg) * a.gs;   // kv head, first q head
    const int heads = min(a.gs, (h + 1) * a.g - h0);
    const int64_t n = length(a, at.b);

    // q of head r: words t W .. t W + W of a row face this thread, eight
    // elements each, in the order that the masks below take a code word apart
    uint32_t qa[2 * W][4];
    float qf, qb;
    {
      const float *q = a.q + at.b * a.ld_q + (int64_t)(h0 + r) * c.dH;
      float big = 0.f, sum = 0.f;
#pragma unroll
      for (int i = 0; i < W; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int d = (t * W + i) * 8 + e;
          const float x = r < heads && d < c.dH ? q[d] : 0.f;
          big = fmaxf(big, fabsf(x));
          sum += x;
        }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // q * up below 2^14, up a power of two (from 2^-115 to 2^113)
      const int ex = max(27, (int)(__float_as_uint(big) >> 23));
      const float up = __uint_as_float((uint32_t)(267 - ex) << 23);
      // codes carry 2^-24
      qf = a.scale * kLog2e * __uint_as_float((uint32_t)min(254, ex + 11) << 23);
      qb = a.scale * kLog2e * sum;
#pragma unroll
      for (int i = 0; i < W; i++) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int d = (t * W + i) * 8 + e;
          x[e] = (r < heads && d < c.dH ? q[d] : 0.f) * up;
          if (e & 1) x[e] *= 0.0625f;      // odd nibbles are met at 16 times their value
        }
        split(x[0], x[4], &qa[2 * i][0], &qa[2 * i][1]);
        split(x[2], x[6], &qa[2 * i][2], &qa[2 * i][3]);
        split(x[1], x[5], &qa[2 * i + 1][0], &qa[2 * i + 1][1]);
        split(x[3], x[7], &qa[2 * i + 1][2], &qa[2 * i + 1][3]);
      }
    }

    float m = -INFINITY, l = 0.f, z = 0.f;
    float o[4 * W][2];
#pragma unroll
    for (int i = 0; i < 4 * W; i++) o[i][0] = o[i][1] = 0.f;
    float *sc = a.scores ? a.scores + (at.b * a.nH + h0 + r) * c.cap : nullptr;

    int64_t next = t0 + warp;
    int put = 0, get = 0;
#pragma unroll
    for (int s = 0; s < kStages - 1; s++) {
      if (next < t1) issue<W>(c, at.b, h, next * TP, (int)min((int64_t)TP, n - next * TP), ring + put * C::kStage);
      asm volatile("cp.async.commit_group;");
      put = put + 1 == kStages ? 0 : put + 1;
      next += kWarps;
    }
    for (int64_t tile = t0 + warp; tile < t1; tile += kWarps) {
      if (next < t1) issue<W>(c, at.b, h, next * TP, (int)min((int64_t)TP, n - next * TP), ring + put * C::kStage);
      asm volatile("cp.async.commit_group;");
      put = put + 1 == kStages ? 0 : put + 1;
      next += kWarps;
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1));
      __syncwarp();
      const uint8_t *ks = ring + get * C::kStage, *vs = ks + C::kCodes, *kgs = vs + C::kCodes;
      const uint8_t *vgs = kgs + 16 * C::kGridStride;
      get = get + 1 == kStages ? 0 : get + 1;
      const int64_t j0 = tile * TP;
      const int cnt = (int)min((int64_t)TP, n - j0);

      // scores of head r against slots 8 nt + 4 e + t
      float s[NT][2];
      {
        const uint8_t *kp = ks + ((r & 1) * 4 + (r >> 1)) * C::kRow + 4 * W * t;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          uint32_t w[W];
          lds<W>(kp + nt * 8 * C::kRow, w);
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < W; i++) {
            const uint32_t x = w[i], y = x >> 8;
            mma(acc, qa[2 * i], x & 0x000f000fu, y & 0x000f000fu);
            mma(acc, qa[2 * i + 1], x & 0x00f000f0u, y & 0x00f000f0u);
          }
          s[nt][0] = (acc[0] + acc[2]) * qf;
          s[nt][1] = (acc[1] + acc[3]) * qf;
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < NT / 2; i++) {
        uint32_t g[4];
        lds<4>(kgs + 4 * (t * C::kGridStride + 4 * i), g);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float &x = s[2 * i + e / 2][e & 1];
          x = fmaf(x, grid_step(g[e]), qb * grid_base(g[e]));
        }
      }
      if (cnt < TP) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            if (8 * nt + 4 * e + t >= cnt) s[nt][e] = -INFINITY;
      }
      if (sc && r < heads) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            if (8 * nt + 4 * e + t < cnt) sc[j0 + 8 * nt + 4 * e + t] = s[nt][e];
      }
#pragma unroll
      for (int nt = 0; nt < NT; nt++) top = fmaxf(top, fmaxf(s[nt][0], s[nt][1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (__any_sync(0xffffffffu, top > m)) {
        const float m1 = fmaxf(m, top), f = m1 > m ? ex2(m - m1) : 1.f;
        m = m1;
        l *= f;
        z *= f;
#pragma unroll
        for (int i = 0; i < 4 * W; i++) {
          o[i][0] *= f;
          o[i][1] *= f;
        }
      }
      // p_j step_j as fp16 pairs: the tile's steps are scaled by a power of two
      // that brings the largest into [2^13, 2^14)
      uint32_t big = 0;
#pragma unroll
      for (int i = 0; i < TP / 32; i++)
        big = max(big, *reinterpret_cast<const uint32_t *>(vgs + 4 * (t * C::kGridStride + r + 8 * i)) << 16 & 0x7fff0000u);
      big = __reduce_max_sync(0xffffffffu, big);
      const int ex = max(13, (int)(big >> 23));
      const float up = __uint_as_float((uint32_t)(267 - ex) << 23);
      const float down = __uint_as_float((uint32_t)min(254, ex + 11) << 23);   // 2^24 / up
      uint32_t pa[KS][4];
      float tl = 0.f, tz = 0.f;
#pragma unroll
      for (int i = 0; i < NT / 2; i++) {
        uint32_t g[4];
        float w[4];
        lds<4>(vgs + 4 * (t * C::kGridStride + 4 * i), g);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float p = ex2(s[2 * i + e / 2][e & 1] - m);
          tl += p;
          tz = fmaf(p, grid_base(g[e]), tz);
          w[e] = p * (grid_step(g[e]) * up);
        }
        split(w[0], w[1], &pa[i][0], &pa[i][1]);
        split(w[2], w[3], &pa[i][2], &pa[i][3]);
      }
      l += tl;
      z += tz;

      // o: column n of an n-tile is element 4 W n + 4 u + v for 16-bit unit u of
      // lane group n's part of the row and nibble v of the unit
      constexpr int VW = W % 2 ? W : W / 2;    // registers a row's part takes (odd W: one unit each)
      uint32_t vw[KS][4][VW];
      {
        const uint8_t *vp = vs + t * C::kRow + 2 * W * r;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
          for (int x = 0; x < 4; x++) {          // slots 16 k + 4 x + t
            const uint8_t *row = vp + (16 * k + 4 * x) * C::kRow;
            if constexpr (W % 2) {
#pragma unroll
              for (int i = 0; i < W; i++) vw[k][x][i] = *reinterpret_cast<const uint16_t *>(row + 2 * i);
            } else {
              lds<VW>(row, vw[k][x]);
            }
          }
      }
#pragma unroll
      for (int u = 0; u < W; u++) {
        float acc[4][4];
#pragma unroll
        for (int v = 0; v < 4; v++) acc[v][0] = acc[v][1] = acc[v][2] = acc[v][3] = 0.f;
        constexpr uint32_t kLow = 0x5410, kHigh = 0x7632;
        const int wi = W % 2 ? u : u / 2;
        const uint32_t sel = W % 2 == 0 && (u & 1) ? kHigh : kLow;
#pragma unroll
        for (int k = 0; k < KS; k++) {
          const uint32_t x = __byte_perm(vw[k][0][wi], vw[k][1][wi], sel), x8 = x >> 8;
          const uint32_t y = __byte_perm(vw[k][2][wi], vw[k][3][wi], sel), y8 = y >> 8;
          mma(acc[0], pa[k], x & 0x000f000fu, y & 0x000f000fu);
          mma(acc[1], pa[k], x & 0x00f000f0u, y & 0x00f000f0u);
          mma(acc[2], pa[k], x8 & 0x000f000fu, y8 & 0x000f000fu);
          mma(acc[3], pa[k], x8 & 0x00f000f0u, y8 & 0x00f000f0u);
        }
#pragma unroll
        for (int v = 0; v < 4; v++) {
          const float f = v & 1 ? down * 0.0625f : down;
          o[4 * u + v][0] = fmaf(acc[v][0] + acc[v][2], f, o[4 * u + v][0]);
          o[4 * u + v][1] = fmaf(acc[v][1] + acc[v][3], f, o[4 * u + v][1]);
        }
      }
      __syncwarp();   // the stage is written again by the next issue
    }
    asm volatile("cp.async.wait_group 0;");

    // the four warps' parts of the segment
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    z += __shfl_xor_sync(0xffffffffu, z, 1);
    z += __shfl_xor_sync(0xffffffffu, z, 2);
    __syncthreads();
    float *part = reinterpret_cast<float *>(sm);            // [kWarps][kHeads][dP + 2]
    {
      float *mine = part + (warp * kHeads + r) * (dP + 2);
#pragma unroll
      for (int u = 0; u < W; u++)
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
          for (int e = 0; e < 2; e++) mine[4 * W * (2 * t + e) + 4 * u + v] = o[4 * u + v][e] + z;
      if (t == 0) {
        mine[dP] = m;
        mine[dP + 1] = l;
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == at.tiles;
    for (int i = threadIdx.x; i < heads * c.dH; i += kThreads) {
      const int hd = i / c.dH, e = i - hd * c.dH;
      const float *x = part + hd * (dP + 2);
      float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) M = fmaxf(M, x[w * kHeads * (dP + 2) + dP]);
#pragma unroll
      for (int w = 0; w < kWarps; w++) {
        const float *y = x + w * kHeads * (dP + 2);
        const float f = y[dP + 1] == 0.f ? 0.f : ex2(y[dP] - M);     // a warp without tiles has l = 0
        L += y[dP + 1] * f;
        O = fmaf(y[e], f, O);
      }
      const int64_t bh = at.b * a.nH + h0 + hd;
      if (whole) {
        a.out[bh * c.dH + e] = O / L;
        if (a.ml && e == 0) a.ml[bh] = make_float2(M, L);
      } else {
        float *dst = a.part + ((int64_t)(2 * blockIdx.x + (t0 == 0)) * kHeads + hd) * (c.dH + 2);
        dst[e] = O;
        if (e == 0) {
          dst[c.dH] = M;
          dst[c.dH + 1] = L;
        }
      }
    }
    __syncthreads();
    u += t1 - t0;
    if (u >= end) break;
    at.tile = 0;
    if (++at.seg == c.nKV * a.hg) {
      at.seg = 0;
      if (threadIdx.x == 0) {      // one reader, so that the threads agree
        do at.tiles = ++at.b < a.B ? (length(a, at.b) + TP - 1) / TP : 1;
        while (at.tiles == 0);
        sh[0] = at.b;
        sh[1] = at.tiles;
      }
      __syncthreads();
      at.b = sh[0];
      at.tiles = sh[1];
      __syncthreads();
    }
  }
}

// Merges the pieces of the segments that run borders cut: block i looks at the
// border before run i and takes the segment if it is the first border inside it.
template <int TILE>
__global__ void __launch_bounds__(kThreads) kv4_attn_merge_kernel(AttnArgs a) {
  pdl_trigger();
  __shared__ int64_t sh[kThreads];
  const Cache &c = a.c;
  pdl_wait();
  const Plan plan = make_plan<TILE>(a, sh);
  const int64_t i = blockIdx.x + 1, u = i * plan.per;
  if (u >= plan.total) return;
  const Place at = find<TILE>(a, u, sh);
  if (at.b < 0 || at.tile == 0 || at.tile > plan.per) return;
  const int h = at.seg / a.hg, h0 = h * a.g + (at.seg % a.hg) * a.gs, hd = blockIdx.y;
  if (hd >= min(a.gs, (h + 1) * a.g - h0)) return;
  const int64_t stride = (int64_t)kHeads * (c.dH + 2);
  const int64_t last = u - at.tile + at.tiles;                       // the segment's end
  const int pieces = 1 + (int)((last - u + plan.per - 1) / plan.per);
  // run i - 1 holds the beginning (slot 1), runs i, i + 1, ... the rest (slot 0)
  const float *base = a.part + hd * (c.dH + 2) + 2 * i * stride;
  auto piece = [&](int p) { return p == 0 ? base - stride : base + 2 * (p - 1) * stride; };
  float M = -INFINITY, L = 0.f;
  const int lane = threadIdx.x & 31;
  for (int p = lane; p < pieces; p += 32) M = fmaxf(M, piece(p)[c.dH]);
  M = warp_max(M);
  for (int p = lane; p < pieces; p += 32) L += piece(p)[c.dH + 1] * ex2(piece(p)[c.dH] - M);
  L = warp_sum(L);
  const int64_t bh = at.b * a.nH + h0 + hd;
  for (int e = threadIdx.x; e < c.dH; e += kThreads) {
    float O = 0.f;
#pragma unroll 4
    for (int p = 0; p < pieces; p++) O = fmaf(piece(p)[e], ex2(piece(p)[c.dH] - M), O);
    a.out[bh * c.dH + e] = O / L;
  }
  if (a.ml && threadIdx.x == 0) a.ml[bh] = make_float2(M, L);
}

// weight_j += sum over the group's q heads of p_j.
constexpr int kWtThreads = 256;
__global__ void __launch_bounds__(kWtThreads) kv4_attn_weights_kernel(AttnArgs a) {
  pdl_trigger();
  const Cache &c = a.c;
  const int h = blockIdx.y, b = blockIdx.z;
  __shared__ float m_s[kMaxGroup], il_s[kMaxGroup];
  pdl_wait();
  const int64_t n = length(a, b), j = (int64_t)blockIdx.x * kWtThreads + threadIdx.x;
  if ((int64_t)blockIdx.x * kWtThreads >= n) return;
  if (threadIdx.x < a.g) {
    const float2 x = a.ml[(int64_t)b * a.nH + h * a.g + threadIdx.x];
    m_s[threadIdx.x] = x.x;
    il_s[threadIdx.x] = 1.f / x.y;
  }
  __syncthreads();
  if (j >= n) return;
  const int64_t row = row_of(c, b, h, j);
  if (row < 0) return;
  const float *sc = a.scores + ((int64_t)b * a.nH + h * a.g) * c.cap + j;
  float w = 0.f;
  for (int i = 0; i < a.g; i++) w = fmaf(ex2(sc[i * c.cap] - m_s[i]), il_s[i], w);
  c.weight[row] += w;
}

// Floats of workspace: the pieces and, where weights are kept, (m, l) and the
// scores.
int64_t part_floats(const Cache &c, int ctas) { return (int64_t)ctas * 2 * kHeads * (c.dH + 2); }
int64_t work_floats(const Cache &c, int B, int nH, int ctas) {
  return part_floats(c, ctas) + (c.weight ? (int64_t)B * nH * (c.cap + 2) : 0);
}

int checked(const char *who, const fcu_kv4 *cache, int B, int nH, bool arrays, Cache *c) {
  FCU_REQUIRE(B >= 0 && B <= 65535, "%s: B=%d", who, B);
  int rc = view(who, cache, B, arrays, c);
  if (rc) return rc;
  FCU_REQUIRE(nH > 0 && nH % c->nKV == 0 && nH / c->nKV <= kMaxGroup, "%s: %d q heads on %d kv heads", who, nH, c->nKV);
  return FCU_OK;
}

// CTAs of the main kernel: all that are resident, or one per tile if the cache
// cannot hold that many.
template <int W>
int plan_ctas(const fcu_ctx *ctx, const Cache &c, int B, int hg) {
  const int64_t tiles = (int64_t)B * c.nKV * hg * ((c.cap + Cfg<W>::kTile - 1) / Cfg<W>::kTile);
  const int64_t all = (int64_t)ctx->num_sms * Cfg<W>::kCtas;
  return (int)(tiles < all ? tiles : all);
}

int plan_ctas(const fcu_ctx *ctx, const Cache &c, int B, int hg) {
  switch (c.rb / 16) {
    case 1: return plan_ctas<1>(ctx, c, B, hg);
    case 2: return plan_ctas<2>(ctx, c, B, hg);
    case 3: return plan_ctas<3>(ctx, c, B, hg);
    case 4: return plan_ctas<4>(ctx, c, B, hg);
    case 6: return plan_ctas<6>(ctx, c, B, hg);
    default: return plan_ctas<8>(ctx, c, B, hg);
  }
}

template <int W>
int launch(fcu_ctx *ctx, const AttnArgs &a) {
  using C = Cfg<W>;
  static bool set[64] = {false};
  if (!set[ctx->device & 63]) {
    FCU_CHECK_CUDA(cudaFuncSetAttribute(kv4_attn_kernel<W>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    set[ctx->device & 63] = true;
  }
  FCU_CHECK_CUDA(launch_pdl(kv4_attn_kernel<W>, dim3(a.ctas), dim3(kThreads), C::kSmem, ctx->stream, a));
  note_launch();
  if (a.ctas > 1) {
    FCU_CHECK_CUDA(launch_pdl(kv4_attn_merge_kernel<C::kTile>, dim3(a.ctas - 1, a.gs), dim3(kThreads), 0, ctx->stream, a));
    note_launch();
  }
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
  const int g = nH / c.nKV;
  return 4 * work_floats(c, B, nH, plan_ctas(ctx, c, B, g > kHeads ? 2 : 1));
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
  a.g = nH / a.c.nKV;
  a.hg = a.g > kHeads ? 2 : 1;
  a.gs = (a.g + a.hg - 1) / a.hg;
  a.ctas = plan_ctas(ctx, a.c, B, a.hg);
  a.scale = (float)scale;
  a.out = out;
  const int64_t need = 4 * work_floats(a.c, B, nH, a.ctas);
  FCU_REQUIRE(work && work_bytes >= need && ((uintptr_t)work & 15) == 0,
              "fcu_kv4_attn: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)need);
  a.part = (float *)work;
  if (a.c.weight) {
    a.ml = (float2 *)(a.part + part_floats(a.c, a.ctas));
    a.scores = (float *)(a.ml + (int64_t)B * nH);
  }
  switch (a.c.rb / 16) {
    case 1: rc = launch<1>(ctx, a); break;
    case 2: rc = launch<2>(ctx, a); break;
    case 3: rc = launch<3>(ctx, a); break;
    case 4: rc = launch<4>(ctx, a); break;
    case 6: rc = launch<6>(ctx, a); break;
    default: rc = launch<8>(ctx, a); break;
  }
  if (rc) return rc;
  if (a.scores) {
    FCU_CHECK_CUDA(launch_pdl(kv4_attn_weights_kernel, dim3(div_up(a.c.cap, kWtThreads), a.c.nKV, B), dim3(kWtThreads),
                              0, ctx->stream, a));
    note_launch();
  }
  return FCU_OK;
}

}  // extern "C"
