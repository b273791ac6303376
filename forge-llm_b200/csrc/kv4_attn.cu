// Attention of one new token per sequence over the 4-bit KV cache
// (fcu_kv4_attn; layout in kv4.cuh).
//
//   s_j = scale (step_j q.c_j + base_j sum q),  p = softmax(s)
//   o_e = sum_j p_j step_j (c_je - 8) + sum_j p_j (base_j + 8 step_j)
//
// (The middle of a row's grid is near the middle of its values.  About base, the two
// sums of o cancel to a small part of either where many slots share the weight.)
//
// One pass over the cache with a running maximum and sum.  The bound is
// reading the cache: a slot of one kv head is 2 (dH / 2 + 4) bytes, and every
// q head of the group uses it while it is on the chip.
//
// Both products run on mma.sync m16n8k32 in integers, the codes as the 16-row
// operand of bytes: a nibble is one AND (for v one LOP3) away from its place, a
// shift for every other, and sums are exact.  The other operand carries fixed-point numbers
// in signed digits of base 256, a head's first two in columns 2t and 2t + 1 (four
// heads to an 8-column tile), so that one thread holds a head's sums side by side:
// q in four digits where a CTA has up to 4 heads, in three (2^-23 of the head's
// largest value) for 8, whose third ones share a tile; p step alike, of the largest
// in the tile.  (fp16 operands of two parts each, codes moved to where their
// subnormals keep their bits, took 65 us where this takes 61, with nine times the
// error over 70001 slots, 6e-6, since the tensor core drops bits when it lines
// products up.  A tcgen05 tile would want the codes expanded in shared memory first, at
// least twice the traffic of the codes themselves; fed from registers the legacy
// pipe is fast enough.)
//
// Work is cut by tiles of slots, not by sequence: the tiles of all (sequence,
// kv head) segments in a row are dealt in equal runs to as many CTAs as the GPU
// holds, so a ragged batch or one long sequence fill it alike.  A segment that
// lies inside one run is finished there; one cut by run borders leaves pieces
// (o, m, l) that a second kernel merges.
//
// A warp takes a tile at a time (128 slots for rows of up to 32 bytes, 64 up to
// 64, 32 beyond: the tile's words and sums stay in registers), k copied a tile
// ahead and v as soon as the last one's has been used, so that one part per warp
// is always on its way and three fit on chip.
//
// Measured on one B200 (copy rate 6.45 TB/s; replayed): 64 sequences of 4096
// slots, 32 / 8 heads of 128, 57 us = 5.1 TB/s (68 us on pages of 16, 73 of 100;
// 8 q heads per kv head 83, 16 146; fcu_attn_decode over the fp32 cache 422 us); one
// sequence of 262000, 12 / 4 heads of 64, 25 us = 3.0 TB/s; 16 x 2047 slots, 16 / 16
// heads of 80, with weights, 25 us.  No pipe is full at 64 x 4096: issue 60 % busy
// (about 1030 instructions a tile of 64 slots), ALU pipe 43 %, tensor pipe 30 %, DRAM at
// 78 % of the copy rate; 11 and 14 warps per SM took the same time.  What bounds it then
// is not known.  Below some 50 MB of cache it is two launches and a few microseconds
// of start and merge.
#include "kv4.cuh"

namespace fcu {
namespace kv4 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kKBufs = 2;      // k tiles on chip, one of them on its way
constexpr float kLog2e = 1.4426950408889634f;
// Powers of two of the scores' scale (kv4_attn_kernel).
constexpr int kDown = 40, kLeastUnit = -126, kMostUnit = 127;

// W: a row is W 16-byte units (dP = 32 W elements).  G: tiles of four q heads.
template <int W, int G>
struct Cfg {
  static constexpr int kTile = W <= 2 ? 128 : W <= 4 ? 64 : 32;        // slots of one warp's step
  static constexpr int kRow = 16 * W;
  static constexpr int kGridStride = kTile / 8 + (kTile > 32 ? 4 : 0);   // words of the grids of slots x, x + 8, ...
  static constexpr int kGrids = 4 * 8 * kGridStride;
  static constexpr int kCodes = kTile * kRow;
  static constexpr int kPart = kCodes + kGrids;                   // a tile's k or v
  static constexpr int kHeads = 4 * G;
  static constexpr int kRing = kWarps * (kKBufs + 1) * kPart;
  static constexpr int kMerge = kWarps * kHeads * (32 * W + 4) * 4;   // the warps' o, m, l at a segment's end
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
  // resident per SM: by registers, and by shared memory (228 KB, 1 KB and the
  // static arrays of each CTA aside).  (One tile of heads over W 4: with 4 a batch
  // of 64 x 4096 on pages of 16 takes 70 us, with 3 73; without pages 61 both.)
  static constexpr int kByRegs = G == 1 ? (W <= 4 ? 4 : 3) : (W <= 4 ? 3 : 2);
  static constexpr int kBySmem = 228 * 1024 / (kSmem + 3 * 1024);
  static constexpr int kCtas = kByRegs < kBySmem ? kByRegs : kBySmem;
};
constexpr int kMaxHeads = 8;           // q heads of one CTA

// What run c leaves for the merge: the segment that begins in it and is cut by
// its end (pieces 0: none).
struct Cut {
  int pieces, heads;
  int64_t bh;            // b * nH + the first head
};

struct AttnArgs {
  const float *q;
  int64_t ld_q;
  Cache c;
  const int32_t *lens;
  int B, nH, g;          // g: q heads per kv head
  int gs, hg;            // q heads of one segment, segments per kv head
  int ctas;              // runs (CTAs of the main kernel)
  int whole;             // every segment is one CTA's: nothing is cut
  int vec;               // q rows and heads start on 16 bytes
  float scale;
  float *out;
  float *part;           // [ctas][2][kMaxHeads][dH + 2]: o, then m (log2 units) and l
  Cut *cuts;             // [ctas]
  float2 *ml;            // [B, nH] where weights are kept: m and l, or of a cut segment (its run's bits, -pieces)
  float *scores;         // [B, nH, cap] in log2 units, where weights are kept
};

__device__ __forceinline__ int64_t length(const AttnArgs &a, int64_t b) {
  const int64_t n = a.lens[b];
  return n < 0 ? 0 : n > a.c.cap ? a.c.cap : n;
}

// What a sequence's segments count for in the cut into runs: their tiles, or one
// where segments stay whole.
template <int TILE>
__device__ __forceinline__ int64_t units(const AttnArgs &a, int64_t b) {
  const int64_t t = (length(a, b) + TILE - 1) / TILE;
  return a.whole && t > 1 ? 1 : t;
}

// The cut into runs: `total` units, `per` of them to a run.  A run is at least a
// tile for every warp of the CTA, unless no segment is that long.
struct Plan {
  int64_t total, per;
};

// A unit's place: sequence, segment of the sequence, unit of the segment.
struct Place {
  int64_t b;
  int seg;
  int64_t tile, tiles;
};

// Block-wide; sh: 2 * kWarps int64.
template <int TILE>
__device__ Plan make_plan(const AttnArgs &a, int64_t *sh) {
  const int segs = a.c.nKV * a.hg;
  int64_t total = 0, longest = 0;
  for (int64_t b = threadIdx.x; b < a.B; b += kThreads) {
    const int64_t t = units<TILE>(a, b);
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

// The place of unit u < total (b = -1 if the lengths have changed since the
// total was taken).  Block-wide, the same for all threads; sh: kThreads int64.
template <int TILE>
__device__ Place find(const AttnArgs &a, int64_t u, int64_t *sh) {
  const int segs = a.c.nKV * a.hg, tid = threadIdx.x;
  int64_t before = 0;
  for (int64_t b0 = 0; b0 < a.B; b0 += kThreads) {
    const int64_t t = b0 + tid < a.B ? units<TILE>(a, b0 + tid) : 0;
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

// make_plan, and find() for the first unit of run `run`, at once for at most
// kThreads sequences (their lengths are read once).  b = -1: the run is empty.
template <int TILE>
__device__ Plan plan_small(const AttnArgs &a, int64_t run, int64_t *sh, Place *at) {
  const int segs = a.c.nKV * a.hg, tid = threadIdx.x;
  const int t = tid < a.B ? (int)units<TILE>(a, tid) : 0;      // at most 2^25 tiles of 2^30 slots
  int64_t x = t;
  int longest = t;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if ((tid & 31) >= o) x += y;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if ((tid & 31) == 31) {
    sh[tid >> 5] = x;
    sh[kWarps + (tid >> 5)] = longest;
  }
  __syncthreads();
  Plan p;
  p.total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) {
    if (w < (tid >> 5)) x += sh[w];
    p.total += sh[w];
    longest = max(longest, (int)sh[kWarps + w]);
  }
  p.total *= segs;
  p.per = max((p.total + a.ctas - 1) / a.ctas, min((int64_t)kWarps, (int64_t)longest));
  const int64_t u = run * p.per;
  __syncthreads();
  if (tid == 0) sh[0] = -1;
  __syncthreads();
  if (u < p.total && (x - t) * segs <= u && u < x * segs) {     // one thread's sequence
    sh[0] = tid;
    sh[1] = u - (x - t) * segs;
    sh[2] = t;
  }
  __syncthreads();
  at->b = sh[0];
  at->tiles = sh[2];
  at->seg = sh[0] < 0 ? 0 : (int)(sh[1] / sh[2]);
  at->tile = sh[0] < 0 ? 0 : sh[1] - at->seg * sh[2];
  __syncthreads();
  return p;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// c += a b, and the same from zero.  A sum c is kept as the bits of the float
// (1.5 2^23 + c) 2^-kDown: kMagic is zero, and of sums below 2^22 one subtraction
// makes c 2^-kDown.
constexpr int kMagic = 0x4b400000 - (kDown << 23);
// SIGNED: a's bytes are.
#define FCU_IMMA "mma.sync.aligned.m16n8k32.row.col.s32."
template <bool SIGNED>
__device__ __forceinline__ void imma(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define FCU_CASE(T)                                                                       \
  asm(FCU_IMMA T ".s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"          \
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])                                    \
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1))
  if constexpr (SIGNED) FCU_CASE("s8");
  else FCU_CASE("u8");
#undef FCU_CASE
}
template <bool SIGNED>
__device__ __forceinline__ void imma0(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define FCU_CASE(T)                                                                       \
  asm(FCU_IMMA T ".s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"      \
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])                                    \
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(kMagic))
  if constexpr (SIGNED) FCU_CASE("s8");
  else FCU_CASE("u8");
#undef FCU_CASE
}
#undef FCU_IMMA
__device__ __forceinline__ float sum_of(int c) { return __int_as_float(c) - __int_as_float(kMagic); }

// 2^e for e in -126 .. 127, and the largest power of two in a float (-127: 2^-126
// or below; 128: not finite).
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23 & 255) - 127; }

// x in signed digits of base 256, a byte each: four of |x| < 2^31 / 1.004 (G 1) or
// the upper three bytes of |x| < 2^23 / 1.004 (G 2), and 2^-kDown times a sum over
// the four digits' sums, the last of which G 2 does not have.
template <int G>
__device__ __forceinline__ uint32_t digits(float x) {
  const uint32_t v = G == 1 ? __float2int_rn(x) : __float2int_rn(x) << 8;
  return (v + 0x80808080u) ^ 0x80808080u;
}
template <int G>
__device__ __forceinline__ float total(int c0, int c1, int c2, int c3) {
  const float low = G == 1 ? fmaf(sum_of(c2), 0x1p8f, sum_of(c3)) : sum_of(c2) * 0x1p8f;
  return fmaf(sum_of(c0), 0x1p24f, fmaf(sum_of(c1), 0x1p16f, low));
}

// Powers of two by which the output's sums over n slots are kept down: 5 to 35.
__device__ __forceinline__ int spare_of(int n) { return 36 - __clz(n); }

// 16 (c - 8) in each byte, c the code in its upper nibble: (x & 0xf0..) ^ 0x80.. in one
// instruction, which the compiler makes two of (64 x 4096 slots 65.6 us, so 63.3).
__device__ __forceinline__ uint32_t middle(uint32_t x) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(y) : "r"(x), "r"(0xf0f0f0f0u), "r"(0x80808080u));
  return y;
}

// Bytes b of four words (sel: b and b + 4 in its nibbles).
__device__ __forceinline__ uint32_t bytes4(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t sel) {
  return __byte_perm(__byte_perm(x0, x1, sel), __byte_perm(x2, x3, sel), 0x5410);
}

// The 8 x 8 matrix of 16-bit elements whose row `lane / 4` the warp holds in
// pairs, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0));
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0));
}

// Shared memory keeps the 16-byte piece c of slot x's row at c ^ swizzle(x), so
// that one piece of eight neighbouring slots lies in all 32 banks, which is what
// ldmatrix reads at a time (odd W: their rows are 4 banks times an odd number
// apart as they are).
template <int W>
__device__ __forceinline__ int swizzle(int x) {
  if constexpr (W == 8) return x & 7;
  else if constexpr (W == 4) return (x >> 1) & 3;
  else if constexpr (W % 2 == 0) return (x >> 2) & 1;
  else return 0;
}
// Where a tile's slot x keeps its grid: those of slots x, x + 8, ... are neighbours.
template <class C>
__device__ __forceinline__ uint32_t grid_at(int x) {
  return 4 * ((x & 7) * C::kGridStride + (x >> 3));
}

// issue() for blocks that sixteen slots may straddle.  (Not inlined, and so the
// cache's geometry goes by value: a reference would put all of it on the stack.)
template <class C, int W>
__device__ __noinline__ void issue_scattered(const int32_t *table, int64_t blocks, int mb, int nKV, int bs,
                                             uint32_t div_mul, int div_shift, const uint8_t *codes,
                                             const uint32_t *grids, int64_t b, int h, int j0, int cnt, uint8_t *part) {
  Cache c;
  c.table = table, c.blocks = blocks, c.mb = mb, c.nKV = nKV, c.bs = bs, c.div_mul = div_mul, c.div_shift = div_shift;
  const int lane = threadIdx.x & 31;
  const uint32_t code_s = (uint32_t)__cvta_generic_to_shared(part), grid_s = code_s + C::kCodes;
  if (cnt == C::kTile && C::kTile <= bs) {
    // a full tile lies in one block or two: `cut` slots and the rest, whose row r1
    // is that of the tile's first slot had it been there
    const int blk = (int)block_index(c, j0), off = j0 - blk * bs, cut = bs - off;
    const int64_t p0 = block_of(c, b, blk), p1 = cut < C::kTile ? block_of(c, b, blk + 1) : p0;
    if (p0 >= 0 && p1 >= 0) {
      const int64_t r0 = (p0 * nKV + h) * bs + off, r1 = (p1 * nKV + h) * bs - cut;
      const uint8_t *s0 = codes + r0 * C::kRow + 16 * lane, *s1 = codes + r1 * C::kRow + 16 * lane;
#pragma unroll
      for (int i = 0; i < C::kTile * W / 32; i++) {
        const int x = i * 32 + lane;
        cp_async16(code_s + 16 * (W % 2 == 0 ? x - x % W + (x % W ^ swizzle<W>(x / W)) : x),
                   (x < cut * W ? s0 : s1) + 512 * i, true);
      }
#pragma unroll
      for (int i = 0; i < C::kTile / 32; i++)
        cp_async4(grid_s + grid_at<C>(lane) + 16 * i, grids + (32 * i + lane < cut ? r0 : r1) + 32 * i + lane, true);
      return;
    }
  }
  for (int x = lane; x < C::kTile; x += 32) {
    const uint32_t at = grid_at<C>(x);
    const int64_t row = x < cnt ? row_of(c, b, h, j0 + x) : -1;
    if (row >= 0 || x >= cnt) cp_async4(grid_s + at, row >= 0 ? grids + row : grids, row >= 0);
    else *reinterpret_cast<uint32_t *>(part + C::kCodes + at) = kNanGrid;
  }
  for (int x = lane; x < C::kTile * W; x += 32) {
    const int j = x / W;
    const int64_t row = j < cnt ? row_of(c, b, h, j0 + j) : -1;
    cp_async16(code_s + 16 * (W % 2 == 0 ? x - x % W + (x % W ^ swizzle<W>(j)) : x),
               row >= 0 ? codes + row * C::kRow + 16 * (x - j * W) : codes, row >= 0);
  }
}

// Starts the copies of one tile's k or v (slots j0 .. j0 + cnt of head h of
// sequence b) into shared memory.  Slots past cnt are zero; those of a bad block
// have NaN grids.  flat: the row of slot 0 where all slots lie in one block, else
// -1.
template <class C, int W>
__device__ __forceinline__ void issue(const Cache &c, const uint8_t *codes, const uint32_t *grids, int64_t flat,
                                      int64_t b, int h, int j0, int cnt, uint8_t *part) {
  const int lane = threadIdx.x & 31;
  const uint32_t code_s = (uint32_t)__cvta_generic_to_shared(part), grid_s = code_s + C::kCodes;
  int64_t row = flat + j0;             // where a full tile's rows are contiguous; -1: they are not
  if (flat < 0) {
    const int blk = (int)block_index(c, j0), off = j0 - blk * c.bs;
    const int64_t p = block_of(c, b, blk);
    row = off + C::kTile <= c.bs && p >= 0 ? (p * c.nKV + h) * c.bs + off : -1;
  }
  if (cnt == C::kTile && row >= 0) {
    const uint8_t *src = codes + row * C::kRow + 16 * lane;
#pragma unroll
    for (int i = 0; i < C::kTile * W / 32; i++) {
      const int x = i * 32 + lane;
      cp_async16(code_s + 16 * (W % 2 == 0 ? x - x % W + (x % W ^ swizzle<W>(x / W)) : x), src + 512 * i, true);
    }
    const uint32_t *g = grids + row + lane;
#pragma unroll
    for (int i = 0; i < C::kTile / 32; i++) cp_async4(grid_s + grid_at<C>(lane) + 16 * i, g + 32 * i, true);
  } else if (c.bs % 16 == 0) {
    // sixteen slots at a time lie in one block: lane i finds the i-th sixteen's
    // first row
    int64_t first = -1;
    if (16 * lane < cnt) first = row_of(c, b, h, j0 + 16 * lane);
    if (cnt == C::kTile && __all_sync(0xffffffffu, first >= 0 || lane >= C::kTile / 16)) {
      // all there: sixteen slots are 16 W pieces in a row
      const uint8_t *p = codes + first * C::kRow;
#pragma unroll
      for (int k = 0; k < C::kTile / 16; k++) {
        const uint64_t at = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(p), k);
        const uint8_t *src = reinterpret_cast<const uint8_t *>(at) + 16 * lane;
#pragma unroll
        for (int i = 0; i < (W + 1) / 2; i++) {
          const int x = i * 32 + lane;
          if (32 * i + 32 <= 16 * W || lane < 16)
            cp_async16(code_s + 16 * (16 * W * k + (W % 2 == 0 ? x - x % W + (x % W ^ swizzle<W>(x / W)) : x)),
                       src + 512 * i, true);
        }
      }
#pragma unroll
      for (int i = 0; i < C::kTile / 32; i++) {
        const int64_t row = __shfl_sync(0xffffffffu, first, 2 * i + (lane >> 4));
        cp_async4(grid_s + grid_at<C>(lane) + 16 * i, grids + row + (lane & 15), true);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < C::kTile / 32; i++) {
      const int x = i * 32 + lane;
      const int64_t row = __shfl_sync(0xffffffffu, first, x >> 4);
      const uint32_t at = grid_at<C>(x);
      const bool on = row >= 0 && x < cnt;
      if (on || x >= cnt) cp_async4(grid_s + at, on ? grids + row + (x & 15) : grids, on);
      else *reinterpret_cast<uint32_t *>(part + C::kCodes + at) = kNanGrid;
    }
#pragma unroll
    for (int i = 0; i < C::kTile * W / 32; i++) {
      const int x = i * 32 + lane, j = x / W;
      const int64_t row = __shfl_sync(0xffffffffu, first, j >> 4);
      const bool on = row >= 0 && j < cnt;
      cp_async16(code_s + 16 * (W % 2 == 0 ? x - x % W + (x % W ^ swizzle<W>(j)) : x),
                 on ? codes + row * C::kRow + 16 * (x - (j & ~15) * W) : codes, on);
    }
  } else {
    issue_scattered<C, W>(c.table, c.blocks, c.mb, c.nKV, c.bs, c.div_mul, c.div_shift, codes, grids, b, h, j0, cnt,
                          part);
  }
}

// 8 x 8 matrices of 16-bit elements, as they lie or transposed: lane i gives row
// i % 8 of matrix i / 8.
template <bool T>
__device__ __forceinline__ void ldsm4(uint32_t p, uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d) {
  if constexpr (T)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(p) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(p) : "memory");
}
template <bool T>
__device__ __forceinline__ void ldsm2(uint32_t p, uint32_t &a, uint32_t &b) {
  if constexpr (T)
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
                 : "=r"(a), "=r"(b) : "r"(p) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(p) : "memory");
}
// The rows of slots 16 k .. 16 k + 16 of a tile: w[e][c] of thread (r, t) is word
// t of piece c of slot 16 k + 8 e + r, or (T) unit r of piece c of slots 2t and
// 2t + 1 of those eight.  off: lane's place for pieces 2c and 2c + 1.
template <int W, bool T>
__device__ __forceinline__ void rows16(uint32_t codes, const uint32_t (&off)[(W + 1) / 2], int k, uint32_t (&w)[2][W]) {
#pragma unroll
  for (int c = 0; c + 1 < W; c += 2)
    ldsm4<T>(codes + off[c / 2] + 16 * k * 16 * W, w[0][c], w[1][c], w[0][c + 1], w[1][c + 1]);
  if constexpr (W % 2) ldsm2<T>(codes + off[W / 2] + 16 * k * 16 * W, w[0][W - 1], w[1][W - 1]);
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

// A warp's thread is (r = lane / 4, t = lane % 4).  It holds head t (and 4 + t)
// at slots r, r + 8, ... of a tile's scores, and in the output head t at the four
// elements that start at 32 c + 4 r of every piece c.
template <int W, int G>
__global__ void __launch_bounds__(kThreads, Cfg<W, G>::kCtas) kv4_attn_kernel(AttnArgs a) {
  using C = Cfg<W, G>;
  constexpr int TP = C::kTile, KS = TP / 16, dP = 32 * W;
  pdl_trigger();
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ int64_t sh[kThreads];
  const Cache &c = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
  uint8_t *kbuf = sm + warp * (kKBufs + 1) * C::kPart, *vbuf = kbuf + kKBufs * C::kPart;
  const uint32_t kbuf_s = (uint32_t)__cvta_generic_to_shared(kbuf), vbuf_s = kbuf_s + kKBufs * C::kPart;
  uint32_t off[(W + 1) / 2];      // this lane's row and piece for ldmatrix
#pragma unroll
  for (int i = 0; i < (W + 1) / 2; i++) {
    const int row = lane & 15;
    off[i] = row * C::kRow + 16 * ((2 * i + (lane >> 4)) ^ swizzle<W>(row));
    if (W % 2 && i == W / 2) off[i] = row * C::kRow + 16 * (W - 1);
  }
  pdl_wait();
  for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x)
    if (length(a, b) == 0)
      for (int i = threadIdx.x; i < a.nH * c.dH; i += kThreads) a.out[b * a.nH * c.dH + i] = 0.f;
  Place at{-1, 0, 0, 0};
  const Plan plan = a.B <= kThreads ? plan_small<TP>(a, blockIdx.x, sh, &at) : make_plan<TP>(a, sh);
  int64_t u = blockIdx.x * plan.per;
  const int64_t end = min(u + plan.per, plan.total);
  Cut cut{0, 0, 0};
  if (a.B > kThreads && u < end) at = find<TP>(a, u, sh);
  while (at.b >= 0 && at.b < a.B) {
    // this run's part [t0, t1) of the segment
    const int t0 = (int)at.tile;
    const int h = at.seg / a.hg, h0 = h * a.g + (at.seg % a.hg) * a.gs;   // kv head, first q head
    const int heads = min(a.gs, (h + 1) * a.g - h0);
    const int n = (int)length(a, at.b);
    const int t1 = a.whole ? (n + TP - 1) / TP : (int)min(at.tiles, at.tile + (end - u));

    int64_t flat = -1;
    if (c.mb == 1) {
      flat = block_of(c, at.b, 0);
      if (flat >= 0) flat = (flat * c.nKV + h) * c.bs;
    }

    // a tile's k and v are copy groups of their own: k one tile ahead, v as soon
    // as the last tile's has been used
    auto issue_k = [&](int tile, int buf) {
      if (tile < t1) issue<C, W>(c, c.k, c.kg, flat, at.b, h, tile * TP, min(TP, n - tile * TP), kbuf + buf * C::kPart);
      asm volatile("cp.async.commit_group;");
    };
    auto issue_v = [&](int tile) {
      if (tile < t1) issue<C, W>(c, c.v, c.vg, flat, at.b, h, tile * TP, min(TP, n - tile * TP), vbuf);
      asm volatile("cp.async.commit_group;");
    };
    int kb = 0;
    issue_k(t0 + warp, 0);
    issue_v(t0 + warp);

    // scale * log2 e * q of head r / 2 against the eight elements of word t of every
    // piece, even ones (the low nibbles) and odd ones: its first digit for even r,
    // the second for odd r, and (qc) the third and fourth or each tile's third
    uint32_t qb[G][W][2], qc[W][2];
    // For head t: its scaled q lie below 2^qe, and their digits stand for 2^(31 - qe) times
    // them.  A sum of codes times digits, below 2^43, is brought down by 2^-kDown before it
    // meets the row's grid, so that no row that the cache holds takes a score out of fp32;
    // scores are kept over unit(), the rest of that scale.  qs: the sum of the scaled q, alike.
    float qs[G];
    int qe[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int head = 4 * g + (r >> 1);
      const float *q = a.q + at.b * a.ld_q + (int64_t)(h0 + head) * c.dH;
      float x[8 * W], big = 0.f;
#pragma unroll
      for (int i = 0; i < 8 * W; i += 4) {
        const int d = 32 * (i / 8) + 8 * t + i % 8;
        if (a.vec) {
          float4 f = {0.f, 0.f, 0.f, 0.f};
          if (head < heads && d < c.dH) f = *reinterpret_cast<const float4 *>(q + d);
          x[i] = f.x, x[i + 1] = f.y, x[i + 2] = f.z, x[i + 3] = f.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) x[i + e] = head < heads && d + e < c.dH ? q[d + e] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 8 * W; i++) big = fmaxf(big, fabsf(x[i]));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // scale log2 e x = (x 2^-e0) sc 2^(e0 + e1): both factors are near 1, whatever q and scale are
      const int e0 = min(126, exponent(big)), e1 = min(126, exponent(a.scale));
      const float near1 = exp2i(-e0), sc = a.scale * exp2i(-e1) * kLog2e;
      const int e2 = min(8, max(-64, exponent(big * near1 * fabsf(sc) * 1.004f) + 1));
      // (below what unit() can be, of use beside keys of 2^100 and more only: fewer digits)
      const int lost = min(64, max(0, kLeastUnit + 31 - kDown - (e0 + e1 + e2)));
      const float up = sc * exp2i((G == 1 ? 31 : 23) - e2 - lost);
      float sum = 0.f;
      const uint32_t sel = r & 1 ? 0x62 : 0x73, sel2 = G == 1 && r & 1 ? 0x40 : 0x51;
#pragma unroll
      for (int i = 0; i < W; i++) {
        uint32_t y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float z = x[8 * i + e] * near1 * up;
          sum += z;
          y[e] = digits<G>(z);
        }
        qb[g][i][0] = bytes4(y[0], y[2], y[4], y[6], sel);
        qb[g][i][1] = bytes4(y[1], y[3], y[5], y[7], sel);
        if (g == 0 || r & 1) {
          qc[i][0] = bytes4(y[0], y[2], y[4], y[6], sel2);
          qc[i][1] = bytes4(y[1], y[3], y[5], y[7], sel2);
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qs[g] = __shfl_sync(0xffffffffu, sum * exp2i((G == 1 ? 0 : 8) - kDown), 8 * t);
      qe[g] = __shfl_sync(0xffffffffu, max(e0 + e1 + e2 + lost, kLeastUnit + 31 - kDown), 8 * t);
    }
    auto unit = [&](int g) { return exp2i(min(qe[g] + kDown - 31, kMostUnit)); };

    // o and z are kept in 2^spare: sums of n weights' values stay below those of the values
    const int spare = spare_of(n);
    // the running maximum (over unit(), as the scores), for head t
    float m[G], l[G], z[G], o[G][4 * W];
#pragma unroll
    for (int g = 0; g < G; g++) {
      m[g] = -INFINITY;
      l[g] = z[g] = 0.f;
#pragma unroll
      for (int i = 0; i < 4 * W; i++) o[g][i] = 0.f;
    }

    for (int tile = t0 + warp; tile < t1; tile += kWarps) {
      const uint8_t *ks = kbuf + kb * C::kPart;
      kb ^= 1;
      issue_k(tile + kWarps, kb);
      asm volatile("cp.async.wait_group 2;");
      __syncwarp();
      const int j0 = tile * TP, cnt = min(TP, n - j0);

      // s[g][2 k + e]: head 4 g + t, slot 16 k + 8 e + r
      float s[G][2 * KS];
      {
        const uint32_t ks_s = kbuf_s + (uint32_t)(ks - kbuf);
        uint32_t gr[2 * KS];
        lds<2 * KS>(ks + C::kCodes + 4 * r * C::kGridStride, gr);
#pragma unroll
        for (int k = 0; k < KS; k++) {      // (two at a time, side by side: 1 % slower)
          uint32_t w[2][W];
          rows16<W, false>(ks_s, off, k, w);
          int acc[G][4], low[4];
#pragma unroll
          for (int i = 0; i < W; i++) {
            const uint32_t x0 = w[0][i], x1 = w[1][i], m4 = 0x0f0f0f0fu;
            const uint32_t cs[4] = {x0 & m4, x1 & m4, x0 >> 4 & m4, x1 >> 4 & m4};
            if (i == 0) imma0<false>(low, cs, qc[0][0], qc[0][1]);
            else imma<false>(low, cs, qc[i][0], qc[i][1]);
#pragma unroll
            for (int g = 0; g < G; g++) {
              if (i == 0) imma0<false>(acc[g], cs, qb[g][0][0], qb[g][0][1]);
              else imma<false>(acc[g], cs, qb[g][i][0], qb[g][i][1]);
            }
          }
#pragma unroll
          for (int g = 0; g < G; g++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const uint32_t gd = gr[2 * k + e];
              const float x = total<G>(acc[g][2 * e], acc[g][2 * e + 1], low[2 * e + (G == 1 ? 0 : g)], low[2 * e + 1]);
              s[g][2 * k + e] = fmaf(x, grid_step(gd), qs[g] * grid_base(gd));
            }
        }
      }
#pragma unroll
      for (int g = 0; g < G; g++)
        if (qe[g] + kDown - 31 > kMostUnit)      // scaled q of 2^118 and more
#pragma unroll
          for (int i = 0; i < 2 * KS; i++) s[g][i] *= exp2i(min(127, qe[g] + kDown - 31 - kMostUnit));
      if (cnt < TP) {
#pragma unroll
        for (int i = 0; i < 2 * KS; i++)
          if (8 * i + r >= cnt)
#pragma unroll
            for (int g = 0; g < G; g++) s[g][i] = -INFINITY;
      }
      if (a.scores) {
#pragma unroll
        for (int g = 0; g < G; g++)
          if (4 * g + t < heads) {
            float *sc = a.scores + (at.b * a.nH + h0 + 4 * g + t) * c.cap + j0 + r;
#pragma unroll
            for (int i = 0; i < 2 * KS; i++)
              if (8 * i + r < cnt) sc[8 * i] = s[g][i] * unit(g);
          }
      }
      float top[G];
      bool grows = false;
#pragma unroll
      for (int g = 0; g < G; g++) {
        top[g] = s[g][0];
#pragma unroll
        for (int i = 1; i < 2 * KS; i++) top[g] = fmaxf(top[g], s[g][i]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top[g] = fmaxf(top[g], __shfl_xor_sync(0xffffffffu, top[g], x));
        grows |= top[g] > m[g];
      }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int g = 0; g < G; g++) {
          const float m1 = fmaxf(m[g], top[g]), f = m1 > m[g] ? ex2((m[g] - m1) * unit(g)) : 1.f;
          m[g] = m1;
          l[g] *= f;
          z[g] *= f;
#pragma unroll
          for (int i = 0; i < 4 * W; i++) o[g][i] *= f;
        }
      }
      // p_j step_j in digits, those of slots r and 8 + r of sixteen side by side,
      // transposed into the operand's columns.  A head's are scaled by a power of
      // two that the largest of them in the tile decides.
      asm volatile("cp.async.wait_group 1;");
      __syncwarp();
      uint32_t pb[G][KS], pc[KS];
      float down[G];
      {
        uint32_t gr[2 * KS];
        lds<2 * KS>(vbuf + C::kCodes + 4 * r * C::kGridStride, gr);
        float tl[G], tz[G], most[G], up[G], qf[G];
#pragma unroll
        for (int g = 0; g < G; g++) tl[g] = tz[g] = most[g] = 0.f, qf[g] = unit(g);
#pragma unroll
        for (int i = 0; i < 2 * KS; i++) {
          const float step = grid_step(gr[i]), mid = fmaf(step, 8.f, grid_base(gr[i]));
#pragma unroll
          for (int g = 0; g < G; g++) {
            const float p = ex2((s[g][i] - m[g]) * qf[g]);
            tl[g] += p;
            tz[g] = fmaf(p, mid, tz[g]);
            s[g][i] = p * step;
            most[g] = fmaxf(most[g], fabsf(s[g][i]));
          }
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
          l[g] += tl[g];
          z[g] = fmaf(tz[g], exp2i(-spare), z[g]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) most[g] = fmaxf(most[g], __shfl_xor_sync(0xffffffffu, most[g], x));
          const int ex = min(252, max(31, (int)(__float_as_uint(most[g] * 1.004f) >> 23)));
          up[g] = __uint_as_float((uint32_t)((G == 1 ? 284 : 276) - ex) << 23);
          down[g] = __uint_as_float((uint32_t)(ex + kDown - 34 - spare) << 23);      // (a sixteenth for middle()'s 16)
        }
#pragma unroll
        for (int k = 0; k < KS; k++) {
          uint32_t y[G][2];
#pragma unroll
          for (int g = 0; g < G; g++) {
            y[g][0] = digits<G>(s[g][2 * k] * up[g]);
            y[g][1] = digits<G>(s[g][2 * k + 1] * up[g]);
            pb[g][k] = transpose8(__byte_perm(y[g][0], y[g][1], 0x6273));
          }
          pc[k] = transpose8(G == 1 ? __byte_perm(y[0][0], y[0][1], 0x4051)
                                    : __byte_perm(__byte_perm(y[0][0], y[0][1], 0x5151),
                                                  __byte_perm(y[G - 1][0], y[G - 1][1], 0x5151), 0x5410));
        }
      }

      // o: rows i and i + 8 of an m-tile are elements v and v + 1 of unit i of
      // piece c (16 bits, four elements), at 32 c + 4 i + v
      uint32_t vw[KS][2][W];
#pragma unroll
      for (int k = 0; k < KS; k++) rows16<W, true>(vbuf_s, off, k, vw[k]);
#pragma unroll
      for (int u = 0; u < W; u++) {
        int acc[G][2][4], low[2][4];
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t cs[2][4];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint32_t x = vw[k + e][0][u], y = vw[k + e][1][u];
            const uint32_t even = __byte_perm(x, y, 0x6240), odd = __byte_perm(x, y, 0x7351);
            cs[0][2 * e] = middle(even << 4), cs[0][2 * e + 1] = middle(even);
            cs[1][2 * e] = middle(odd << 4), cs[1][2 * e + 1] = middle(odd);
          }
#pragma unroll
          for (int x = 0; x < 2; x++) {
            if (k == 0) imma0<true>(low[x], cs[x], pc[0], pc[1]);
            else imma<true>(low[x], cs[x], pc[k], pc[k + 1]);
#pragma unroll
            for (int g = 0; g < G; g++) {
              if (k == 0) imma0<true>(acc[g][x], cs[x], pb[g][0], pb[g][1]);
              else imma<true>(acc[g][x], cs[x], pb[g][k], pb[g][k + 1]);
            }
          }
        }
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
          for (int x = 0; x < 2; x++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const float v = total<G>(acc[g][x][2 * e], acc[g][x][2 * e + 1], low[x][2 * e + (G == 1 ? 0 : g)],
                                       low[x][2 * e + 1]);
              o[g][4 * u + 2 * x + e] = fmaf(v, down[g], o[g][4 * u + 2 * x + e]);
            }
      }
      __syncwarp();
      issue_v(tile + kWarps);
    }
    asm volatile("cp.async.wait_group 0;");

    // the four warps' parts of the segment
    __syncthreads();
    float *part = reinterpret_cast<float *>(sm);            // [kWarps][kHeads][dP + 4]: o, m, l
#pragma unroll
    for (int g = 0; g < G; g++) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        l[g] += __shfl_xor_sync(0xffffffffu, l[g], x);
        z[g] += __shfl_xor_sync(0xffffffffu, z[g], x);
      }
      float *mine = part + (warp * C::kHeads + 4 * g + t) * (dP + 4);
#pragma unroll
      for (int i = 0; i < W; i++)
        *reinterpret_cast<float4 *>(mine + 32 * i + 4 * r) =
            make_float4(o[g][4 * i] + z[g], o[g][4 * i + 1] + z[g], o[g][4 * i + 2] + z[g], o[g][4 * i + 3] + z[g]);
      // (m in log2 units from here on)
      if (r == 0) *reinterpret_cast<float2 *>(mine + dP) = make_float2(m[g] * unit(g), l[g] * exp2i(-spare));
    }
    __syncthreads();
    const bool whole = a.whole || (t0 == 0 && t1 == at.tiles);
    const int64_t bh0 = at.b * a.nH + h0;
    if (t0 == 0 && !whole)
      cut = Cut{1 + (int)((at.tiles - t1 + plan.per - 1) / plan.per), heads, bh0};
    if (a.ml && t0 == 0 && !whole && threadIdx.x < heads)
      a.ml[bh0 + threadIdx.x] = make_float2(__int_as_float(blockIdx.x), -(float)cut.pieces);
    for (int i = threadIdx.x; i < heads * (dP / 4); i += kThreads) {
      const int hd = i / (dP / 4), e = 4 * (i - hd * (dP / 4));
      const float *x = part + hd * (dP + 4);
      float M = -INFINITY, L = 0.f;
      float4 O = {0.f, 0.f, 0.f, 0.f};
      float2 ml[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; w++) {
        ml[w] = *reinterpret_cast<const float2 *>(x + w * C::kHeads * (dP + 4) + dP);
        if (ml[w].y != 0.f) M = fmaxf(M, ml[w].x);       // a warp without tiles has l = 0
      }
#pragma unroll
      for (int w = 0; w < kWarps; w++) {
        const float4 y = *reinterpret_cast<const float4 *>(x + w * C::kHeads * (dP + 4) + e);
        const float f = ml[w].y == 0.f ? 0.f : ex2(ml[w].x - M);
        L += ml[w].y * f;
        O.x = fmaf(y.x, f, O.x), O.y = fmaf(y.y, f, O.y), O.z = fmaf(y.z, f, O.z), O.w = fmaf(y.w, f, O.w);
      }
      float *dst;
      if (whole) {
        const float inv = 1.f / L;
        O.x *= inv, O.y *= inv, O.z *= inv, O.w *= inv;
        dst = a.out + (bh0 + hd) * c.dH;
        if (a.ml && e == 0) a.ml[bh0 + hd] = make_float2(M, L);
      } else {
        dst = a.part + ((int64_t)(2 * blockIdx.x + (t0 == 0)) * kMaxHeads + hd) * (c.dH + 2);
        if (e == 0) dst[c.dH] = M, dst[c.dH + 1] = L;
      }
      if (e < c.dH) *reinterpret_cast<float2 *>(dst + e) = make_float2(O.x, O.y);            // dH is even
      if (e + 2 < c.dH) *reinterpret_cast<float2 *>(dst + e + 2) = make_float2(O.z, O.w);
    }
    __syncthreads();
    u += a.whole ? 1 : t1 - t0;
    if (u >= end) break;
    at.tile = 0;
    if (++at.seg == c.nKV * a.hg) {
      at.seg = 0;
      if (threadIdx.x == 0) {      // one reader, so that the threads agree
        do at.tiles = ++at.b < a.B ? units<TP>(a, at.b) : 1;
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
  if (threadIdx.x == 0 && !a.whole) a.cuts[blockIdx.x] = cut;
}

// The (m, l) of a head whose segment begins in run `run` and has `pieces`
// pieces: run `run` holds the first (slot 1), runs run + 1, ... the rest (slot
// 0).  By a warp.
struct Pieces {
  const float *first;
  int64_t stride;
  __device__ Pieces(const AttnArgs &a, int run, int hd) {
    stride = (int64_t)kMaxHeads * (a.c.dH + 2);
    first = a.part + (2 * (int64_t)run + 1) * stride + hd * (a.c.dH + 2);
  }
  __device__ const float *operator[](int p) const { return first + (p == 0 ? 0 : 2 * p - 1) * stride; }
  __device__ float2 ml(int pieces, int dH) const {
    const int lane = threadIdx.x & 31;
    float M = -INFINITY, L = 0.f;
    for (int p = lane; p < pieces; p += 32) {
      const float m = (*this)[p][dH], l = (*this)[p][dH + 1];
      const float m1 = fmaxf(M, m);
      L = (L == 0.f ? 0.f : L * ex2(M - m1)) + l * ex2(m - m1);
      M = m1;
    }
    const float top = warp_max(M);
    return make_float2(top, warp_sum(L == 0.f ? 0.f : L * ex2(M - top)));
  }
};

// What is left when all runs are done.  The first ctas - 1 blocks merge the
// pieces of the segments that begin in a run and go past its end: block i those
// of run i, a warp to a head, if they are at most kFewPieces; a segment of more
// pieces has as many runs to itself, and block i + d takes its d-th head, all
// warps together.  Where weights are kept the other blocks add them up,
// weight_j += sum over the group's q heads of p_j, kWtSlots slots each.
// (kFewPieces is at least kMaxHeads, so that the blocks are the segment's own.  32768
// slots, a warp to a head and all warps to one: 18 pieces a segment 36.7 and 34.2 us, 37
// pieces 28.5 and 24.5; 9 pieces 35.4 and 34.8.)
constexpr int kFewPieces = 12;
constexpr int kFinishThreads = 256;
constexpr int kFinishWarps = kFinishThreads / 32;
constexpr int kWtSlots = 1024;
template <int W, bool VEC>
__global__ void __launch_bounds__(kFinishThreads) kv4_attn_finish_kernel(AttnArgs a) {
  pdl_trigger();
  __shared__ float o_s[kFinishWarps][32 * W];
  __shared__ float m_s[kMaxGroup], il_s[kMaxGroup];
  const Cache &c = a.c;
  const int dH = c.dH, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, merges = a.whole ? 0 : a.ctas - 1;
  pdl_wait();
  if (blockIdx.x < merges) {
    Cut cut{0, 0, 0};
    const int run0 = (int)blockIdx.x - lane;
    if (lane < kMaxHeads && run0 >= 0) cut = a.cuts[run0];
    // (nothing is written elsewhere whatever another call made of the workspace)
    if (cut.heads < 0 || cut.heads > kMaxHeads || cut.bh < 0 || cut.bh + cut.heads > (int64_t)a.B * a.nH)
      cut.pieces = 0;
    const bool mine = lane == 0 ? cut.pieces > 0 : cut.pieces > kFewPieces && lane < cut.heads;
    const uint32_t who = __ballot_sync(0xffffffffu, mine);
    if (!who) return;
    const int d = __ffs(who) - 1, run = (int)blockIdx.x - d;
    cut.pieces = __shfl_sync(0xffffffffu, cut.pieces, d);
    cut.heads = __shfl_sync(0xffffffffu, cut.heads, d);
    cut.bh = __shfl_sync(0xffffffffu, cut.bh, d);
    const int pieces = min(cut.pieces, a.ctas - run);
    const bool few = cut.pieces <= kFewPieces;
    // few: a warp takes a head; else each warp its share of the pieces of head d.
    // Everything of a piece is asked for at once.
    const int hd = few ? warp : d;
    if (few && hd >= cut.heads) return;
    const Pieces part(a, run, hd);
    float M = -INFINITY, L = 0.f, O[W];
#pragma unroll
    for (int i = 0; i < W; i++) O[i] = 0.f;
    constexpr int kBatch = W <= 2 ? 8 : W <= 4 ? 4 : 2;
    const int stride = few ? 1 : kFinishWarps;
    for (int p0 = few ? 0 : warp; p0 < pieces; p0 += kBatch * stride) {
      float m[kBatch], l[kBatch], o[kBatch][W];
#pragma unroll
      for (int k = 0; k < kBatch; k++) {
        const int p = p0 + k * stride;
        const float *x = part[min(p, pieces - 1)];
        m[k] = p < pieces ? x[dH] : -INFINITY;
        l[k] = p < pieces ? x[dH + 1] : 0.f;
#pragma unroll
        for (int i = 0; i < W; i++) o[k][i] = p < pieces && lane + 32 * i < dH ? x[lane + 32 * i] : 0.f;
      }
      float m1 = M;
#pragma unroll
      for (int k = 0; k < kBatch; k++) m1 = fmaxf(m1, m[k]);
      const float f0 = L == 0.f ? 0.f : ex2(M - m1);
      M = m1;
      L *= f0;
#pragma unroll
      for (int i = 0; i < W; i++) O[i] *= f0;
#pragma unroll
      for (int k = 0; k < kBatch; k++) {
        const float f = p0 + k * stride < pieces ? ex2(m[k] - m1) : 0.f;
        L = fmaf(l[k], f, L);
#pragma unroll
        for (int i = 0; i < W; i++) O[i] = fmaf(o[k][i], f, O[i]);
      }
    }
    float *out = a.out + (cut.bh + hd) * dH;
    if (few) {
#pragma unroll
      for (int i = 0; i < W; i++)
        if (lane + 32 * i < dH) out[lane + 32 * i] = O[i] / L;
      return;
    }
    if (lane == 0) {
      m_s[warp] = M;
      il_s[warp] = L;
    }
#pragma unroll
    for (int i = 0; i < W; i++) o_s[warp][lane + 32 * i] = O[i];
    __syncthreads();
    M = m_s[0];
    for (int w = 1; w < kFinishWarps; w++) M = fmaxf(M, m_s[w]);
    L = 0.f;
    for (int w = 0; w < kFinishWarps; w++) L += il_s[w] * ex2(m_s[w] - M);
    for (int e = threadIdx.x; e < dH; e += kFinishThreads) {
      float o = 0.f;
#pragma unroll
      for (int w = 0; w < kFinishWarps; w++) o = fmaf(o_s[w][e], ex2(m_s[w] - M), o);
      out[e] = o / L;
    }
    return;
  }
  const int64_t i = blockIdx.x - merges, chunks = (c.cap + kWtSlots - 1) / kWtSlots;
  const int64_t bk = i / chunks, j0 = (i - bk * chunks) * kWtSlots, b = bk / c.nKV;
  const int h = (int)(bk - b * c.nKV);
  const int64_t n = length(a, b);
  if (j0 >= n) return;
  // what does not wait for (m, l) is asked for first
  constexpr int kPer = kWtSlots / kFinishThreads, kAhead = 4;
  static_assert(kPer == 4, "");
  const float *sc = a.scores + (b * a.nH + h * a.g) * c.cap + j0;
  // VEC: a thread's four slots are neighbours, 16 aligned bytes of scores and weight
  constexpr int kStep = VEC ? 1 : kFinishThreads;
  const int mine = VEC ? 4 * threadIdx.x : threadIdx.x;
  float w[kPer] = {0.f, 0.f, 0.f, 0.f}, old[kPer], s[kAhead][kPer];
  int64_t row[kPer];
  auto load = [&](float (&x)[kPer], const float *p) {
    if constexpr (VEC) {
      const float4 f = row[0] >= 0 ? *reinterpret_cast<const float4 *>(p) : float4{0.f, 0.f, 0.f, 0.f};
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < kPer; k++) x[k] = row[k] >= 0 ? p[k * kStep] : 0.f;
    }
  };
#pragma unroll
  for (int k = 0; k < kPer; k++) {
    const int64_t j = j0 + mine + k * kStep;
    row[k] = VEC && k > 0 ? (j < n && row[0] >= 0 ? row[0] + k : -1) : j < n ? row_of(c, b, h, j) : -1;
  }
  if constexpr (VEC) {
    load(old, c.weight + row[0]);
  } else {
#pragma unroll
    for (int k = 0; k < kPer; k++) old[k] = row[k] >= 0 ? c.weight[row[k]] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < kAhead; i++)
    if (i < a.g) load(s[i], sc + i * c.cap + mine);
  for (int hd = warp; hd < a.g; hd += kFinishWarps) {
    float2 x = a.ml[b * a.nH + h * a.g + hd];
    // a cut segment's: the run it begins in, and minus its pieces
    if (x.y < 0.f) {
      const int run = min(max(__float_as_int(x.x), 0), a.ctas - 1), pieces = min((int)-x.y, a.ctas - run);
      x = Pieces(a, run, hd % a.gs).ml(pieces, dH);
    }
    if (lane == 0) {
      m_s[hd] = x.x;
      il_s[hd] = exp2i(-spare_of((int)n)) / x.y;      // (l is kept as o is)
    }
  }
  __syncthreads();
  for (int hd = 0; hd < a.g; hd += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; i++)
      if (hd + i < a.g) {
        const float m = m_s[hd + i], il = il_s[hd + i];
#pragma unroll
        for (int k = 0; k < kPer; k++) w[k] = fmaf(ex2(s[i][k] - m), il, w[k]);
        if (hd + i + kAhead < a.g) load(s[i], sc + (hd + i + kAhead) * c.cap + mine);
      }
  }
  if (VEC && row[3] >= 0) {
    *reinterpret_cast<float4 *>(c.weight + row[0]) =
        make_float4(old[0] + w[0], old[1] + w[1], old[2] + w[2], old[3] + w[3]);
  } else {
#pragma unroll
    for (int k = 0; k < kPer; k++)
      if (row[k] >= 0) c.weight[row[k]] = old[k] + w[k];
  }
}

// How the heads are dealt: q heads per kv head, segments per kv head (a CTA
// takes at most 8 heads), q heads of a segment, and the CTAs.
struct Heads {
  int g, hg, gs, ctas, whole;
};

// Floats of workspace: the cuts, the pieces and, where weights are kept, (m, l)
// and the scores.
int64_t part_floats(const Cache &c, const Heads &p) {
  return p.whole ? 0 : (int64_t)p.ctas * (2 * kMaxHeads * (c.dH + 2) + sizeof(Cut) / 4);
}
int64_t ml_floats(int B, int nH) { return (2 * (int64_t)B * nH + 3) & ~(int64_t)3; }
int64_t work_floats(const Cache &c, int B, int nH, const Heads &p) {
  return part_floats(c, p) + (c.weight ? ml_floats(B, nH) + (int64_t)B * nH * c.cap : 0);
}

int checked(const char *who, const fcu_kv4 *cache, int B, int nH, bool arrays, Cache *c) {
  FCU_REQUIRE(B >= 0 && B <= 65535, "%s: B=%d", who, B);
  int rc = view(who, cache, B, arrays, c);
  if (rc) return rc;
  FCU_REQUIRE(nH > 0 && nH % c->nKV == 0 && nH / c->nKV <= kMaxGroup, "%s: %d q heads on %d kv heads", who, nH, c->nKV);
  return FCU_OK;
}

// CTAs of the main kernel: all that are resident, or one per tile if the cache
// cannot hold that many.  A cache of at most kWholeTiles tiles per sequence
// whose segments are all resident at once gives each a CTA of its own: its two
// steps per warp cost less than the second kernel that would merge pieces.  (Full caches
// of 8 tiles, whole and merged: 1 x 1024 slots of 12 / 4 heads of 64 6.1 and 7.1 us, 1 x
// 512 of 32 / 8 heads of 128 6.4 and 7.3, 16 x 512 9.3 and 10.5, 64 x 512 13.5 and 21.8.
// Of 16 tiles: 8.7 and 7.1, 9.0 and 8.4, 14.5 and 12.9, but 20.2 and 25.8.)
constexpr int kWholeTiles = 8;
template <int W, int G>
void plan_ctas(const fcu_ctx *ctx, const Cache &c, int B, Heads *p) {
  using C = Cfg<W, G>;
  const int64_t tiles = (c.cap + C::kTile - 1) / C::kTile, segs = (int64_t)B * c.nKV * p->hg;
  const int64_t all = (int64_t)ctx->num_sms * C::kCtas;
  p->whole = tiles <= kWholeTiles && segs <= all;
  p->ctas = (int)(p->whole ? segs : segs * tiles < all ? segs * tiles : all);
}

template <int W, int G>
int launch(fcu_ctx *ctx, const AttnArgs &a) {
  using C = Cfg<W, G>;
  static bool set[64] = {false};
  if (!set[ctx->device & 63]) {
    FCU_CHECK_CUDA(cudaFuncSetAttribute(kv4_attn_kernel<W, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    set[ctx->device & 63] = true;
  }
  FCU_CHECK_CUDA(launch_pdl(kv4_attn_kernel<W, G>, dim3(a.ctas), dim3(kThreads), C::kSmem, ctx->stream, a));
  note_launch();
  const int64_t sums = a.scores ? (int64_t)a.B * a.c.nKV * ((a.c.cap + kWtSlots - 1) / kWtSlots) : 0;
  const int64_t blocks = (a.whole ? 0 : a.ctas - 1) + sums;
  if (blocks > 0) {
    const bool vec = a.scores && a.c.cap % 4 == 0 && a.c.bs % 4 == 0 && ((uintptr_t)a.c.weight & 15) == 0;
    FCU_CHECK_CUDA(launch_pdl(vec ? kv4_attn_finish_kernel<W, true> : kv4_attn_finish_kernel<W, false>,
                              dim3((unsigned)blocks), dim3(kFinishThreads), 0, ctx->stream, a));
    note_launch();
  }
  return FCU_OK;
}

// f(W, G) for a cache's row width and a segment's heads
#define FCU_KV4_WIDTHS(f, rb, gs)                                      \
  switch ((rb) / 16 * 2 + ((gs) > 4)) {                                \
    case 2: f(1, 1); break;                                            \
    case 3: f(1, 2); break;                                            \
    case 4: f(2, 1); break;                                            \
    case 5: f(2, 2); break;                                            \
    case 6: f(3, 1); break;                                            \
    case 7: f(3, 2); break;                                            \
    case 8: f(4, 1); break;                                            \
    case 9: f(4, 2); break;                                            \
    case 12: f(6, 1); break;                                           \
    case 13: f(6, 2); break;                                           \
    case 16: f(8, 1); break;                                           \
    default: f(8, 2); break;                                           \
  }

Heads plan_heads(const fcu_ctx *ctx, const Cache &c, int B, int nH) {
  Heads p;
  p.g = nH / c.nKV;
  p.hg = p.g > kMaxHeads ? 2 : 1;
  p.gs = (p.g + p.hg - 1) / p.hg;
#define FCU_CASE(W, G) plan_ctas<W, G>(ctx, c, B, &p)
  FCU_KV4_WIDTHS(FCU_CASE, c.rb, p.gs)
#undef FCU_CASE
  return p;
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
  return 4 * work_floats(c, B, nH, plan_heads(ctx, c, B, nH));
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
  FCU_REQUIRE(((uintptr_t)out & 7) == 0, "fcu_kv4_attn: out is not 8-byte aligned");
  a.q = q;
  a.ld_q = ld_q;
  a.lens = seq_lens;
  a.B = B;
  a.nH = nH;
  const Heads p = plan_heads(ctx, a.c, B, nH);
  a.g = p.g;
  a.hg = p.hg;
  a.gs = p.gs;
  a.ctas = p.ctas;
  a.whole = p.whole;
  a.vec = ld_q % 4 == 0 && a.c.dH % 4 == 0 && ((uintptr_t)q & 15) == 0;
  a.scale = (float)scale;
  a.out = out;
  FCU_REQUIRE(!a.c.weight || (double)B * a.c.nKV * (a.c.cap / kWtSlots + 1) < 1e9,
              "fcu_kv4_attn: the cache is too large");
  const int64_t need = 4 * work_floats(a.c, B, nH, p);
  FCU_REQUIRE(need == 0 || (work && work_bytes >= need && ((uintptr_t)work & 15) == 0),
              "fcu_kv4_attn: workspace of %lld bytes, %lld needed", (long long)work_bytes, (long long)need);
  a.cuts = (Cut *)work;
  a.part = (float *)(a.cuts + a.ctas);
  FCU_REQUIRE(out + (int64_t)B * nH * a.c.dH <= q || q + (B - 1) * ld_q + (int64_t)nH * a.c.dH <= out,
              "fcu_kv4_attn: out overlaps q");
  if (a.c.weight) {
    a.ml = (float2 *)((float *)work + part_floats(a.c, p));
    a.scores = (float *)a.ml + ml_floats(B, nH);
  }
#define FCU_CASE(W, G) rc = launch<W, G>(ctx, a)
  FCU_KV4_WIDTHS(FCU_CASE, a.c.rb, a.gs)
#undef FCU_CASE
  if (rc) return rc;
  return FCU_OK;
}

}  // extern "C"
