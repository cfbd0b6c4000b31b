// Shared-prefix decode attention on the tensor cores: bf16/fp16, head size 64 or 128.
//
// Two launches: parts_kernel leaves partial results, join_kernel joins them.
//
// parts_kernel works on units, of two kinds:
//   shared: the query rows of a group that use one KV head (sequence, then head), cut into
//           tiles, against the group's shared tokens;
//   own:    the R query rows of a sequence that use one KV head against the tokens behind
//           the shared ones.
// The tokens of a unit are cut into chunks of 128.  The chunks of all units, shared ones
// first, are laid end to end on a scale of costs (see Costs), and CTA c of the persistent
// grid takes the chunks that begin in [c T / C, (c + 1) T / C) of the total T.  The part of
// a unit inside a CTA's range is a segment.  CTAs on compute-bound shared units run beside
// CTAs on memory-bound own units.
//   warps 0-3, 4-7   two softmax warpgroups ("streams"), a query row per thread;
//   warps 8, 10      TMA producers, 128-byte swizzled tiles: Q and K pages, V pages (a box
//                    takes some 70 cycles to issue, and a page of 16 tokens is 4 KB of K);
//   warp 11          the plan that join_kernel finds the partials by;
//   warp 9           tcgen05 issuer: S = Q K^T (both in shared memory), O += P V (P in
//                    TMEM over S's columns, V as an MN-major operand, so no transpose).
// TMEM: S and O of both streams, 4 x 128 fp32 columns at head size 128 = all 512.
//
// Items: (chunk, row tile of 128) products, numbered through the CTA's range; item i belongs
// to stream i & 1, so the softmax of one item runs under the products of the next, also
// across segments.  The issuer runs S two items ahead of P V.  Segments with up to 128 rows
// have one item per chunk: their chunks alternate between the streams, and each stream
// leaves a partial of its own.  Segments with 256 rows ("wide") have two items per chunk,
// which halves the K/V traffic per row.  Tiles are wide when a group has more than 128 rows
// (measured with narrow tiles against: 4 groups of 256 rows x 8192 tokens 78 us and 72, 256
// rows x 512 tokens 24.9 and 23.2).
//
// The running maximum is only raised when it would grow by more than 8 (log2, fp16: 4): weights
// above 1 are harmless in 16 bits, and O is then rarely rescaled.  Rounded to 16 bits: the
// weights P, as a tensor-core operand (a relative 2^-9 or 2^-12 each, at random: the plain
// 64-bit result is off by up to 40% more than with fp32 weights; the weights of paged_decode are
// rounded alike, and two products of halves would double the tensor cores' work); the maximum,
// the sum, S and O are fp32.  fp16 has few exponents: its weights are 2^8 times as large (2^12
// at most, finite up to scores of 2^26), so that one of 2^-22 of the greatest still has all its
// bits and the smaller ones are off by 2^-33 of the greatest at most.
//
// Bound: HBM where few rows share a token (8 sequences of 131 thousand: 105 us for 541 MB, 79%
// of a plain copy's rate with start-up and join); with 128 sequences the chain of product,
// softmax and product (120 us, of which the tensor cores need 42), some 2,100 cycles per item
// of 128 x 128.  (Device times of captured calls; a call from the host takes 115 and 130 us.)
// Before the first scores some 12 us pass, on code and tables from HBM.
#pragma once

#include "shared_prefix.cuh"

namespace llmc {
namespace prefix {
namespace tc {

constexpr int kChunk = 128;        // tokens of a chunk (MMA N of S, K of P V)
constexpr int kRing = 8;            // segments the producer may be ahead
constexpr int kThreads = 384;      // two softmax warpgroups, one for the producer and the issuer
// Of the weights, log2: how far the maximum may lag behind, and their scale.
template <typename T>
constexpr float kLag = __is_same(T, __half) ? 4.f : 8.f;
template <typename T>
constexpr float kScale = __is_same(T, __half) ? 8.f : 0.f;

struct TcParams {
  Params p;
  int4* plan;          // [B][Hkv], see below
  int32_t* heads;      // tables_kernel's totals
  int32_t* tables;     // the tables, where they are in global memory
  float* own_o;        // partials of own units, beside p.part_o / part_lse of shared ones
  float* own_lse;
  int nb;              // sequences of a Q tile: nb * R <= 128 rows
  int rs;              // rows of a shared slot
  int ctas;            // grid of parts_kernel
};

// The plan: an int4 per (sequence, KV head), where join_kernel finds its partials:
// {first shared slot, first own slot, shared slots | row << 16 | wide << 31, own slots}.

// Partials of segment (unit u, CTA c): slots 2 (u + c) and 2 (u + c) + 1, unique because
// units and ranges both ascend.  A slot is [D / 4][rows][4] fp32, so that the lanes of a
// warp (rows) store 16-byte pieces side by side.

// This kernel's code is fetched anew in every decode step (the weights that stream between two
// launches push it out of the caches), some 200 cycles for every eight instructions.  So what
// is not in an inner loop is kept small: loops are not unrolled, helpers are not inlined.

// x / n for x >= 0, n > 0: the estimate is off by a few at most (24-bit mantissas).
__device__ __noinline__ int quot(int x, int n) {
  int q = (int)(__int2float_rz(x) * __frcp_rn((float)n));
  int r = x - q * n;
#pragma unroll 1
  while (r < 0) {
    --q;
    r += n;
  }
#pragma unroll 1
  while (r >= n) {
    ++q;
    r -= n;
  }
  return q;
}

// Waits for the barrier's phase of this parity.  Gives up after kWaits attempts (each lets the
// warp sleep for up to microseconds), or when another warp has: the flag and the status word
// say so, and every later wait returns at once.
constexpr int kWaits = 1 << 20;
__device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                     int* status) {
#pragma unroll 1
  for (int i = 0; !mbar_try_wait(bar, parity); ++i) {
    if (*abort_flag) break;
    if (i == kWaits) {
      *abort_flag = 1;
      atomicOr(status, kStatusWaitTimeout);
    }
  }
}

// What the chunks cost, in units of some 450 cycles: a chunk of 128 rows at most 6 (K and V
// of 64 KB at a fair share of the bandwidth are 2700 cycles), a chunk of a wide tile 10; a unit
// 4 more, for the turn-over of a stream, and 1 per 16 rows that leave partials (fitted to the
// CTAs' end times).  With few chunks for the CTAs every chunk is 1.
struct Cost {
  int chunk, unit;
  // of a unit of n chunks: chunk j begins at j * chunk, the unit's own cost is behind the last
  __device__ __forceinline__ int size(int n) const { return n ? n * chunk + unit : 0; }
  // the first chunk that begins at x or later
  __device__ __forceinline__ int chunk_from(int x) const {
    return x <= 0 ? 0 : quot(x + chunk - 1, chunk);
  }
};
struct Costs {
  bool few;
  int narrow;   // rows of a narrow tile
  __device__ __forceinline__ void set(int chunks, int narrow_, int ctas) {
    // Otherwise a CTA's share, 12 at least, exceeds any chunk's cost: no CTA between a unit's
    // first and last one goes without a chunk of it (and leaves its slots unwritten).
    few = chunks < 2 * ctas;
    narrow = narrow_;
  }
  // of the units of a group with so many rows
  __device__ __forceinline__ Cost shared(int rows) const {
    if (few) return {1, 0};
    return {rows > narrow ? 10 : 6, 4 + (min(rows, 2 * narrow) >> 4)};
  }
  __device__ __forceinline__ Cost own() const { return {few ? 1 : 6, few ? 0 : 4}; }
};

// How the total cost is dealt to C CTAs.
struct Split {
  int C, total, q, r;
  __device__ __forceinline__ void set(int total_, int ctas) {
    total = total_;
    // With fewer chunks than CTAs the first ones have one each: no CTA between a unit's first
    // and last is without a part of it.
    C = min(ctas, total);
    q = C ? quot(total, C) : 0;
    r = total - q * C;
  }
  __device__ __forceinline__ int start(int c) const {   // floor(c total / C), c <= C
    return c * q + quot(c * r, C);
  }
  __device__ __noinline__ int owner(int x) const {   // the last c with start(c) <= x
    const long long ec = (long long)(x + 1) * C;        // start(c) <= x  <=>  c total < (x + 1) C
    int c = min(C - 1, (int)((float)x * (float)C * __frcp_rn((float)total)));
#pragma unroll 1
    while (c + 1 < C && (long long)(c + 1) * total < ec) ++c;
#pragma unroll 1
    while (c > 0 && (long long)c * total >= ec) --c;
    return c;
  }
};

// ---- tcgen05 -------------------------------------------------------------------
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t addr) {
  // 128-byte swizzle, rows of 128 bytes: 8-row groups 1024 bytes apart.
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) |
         (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t addr, int box, int halves) {
  // 128-byte swizzle, 64 contiguous N elements per row (a token), laid out [box][half][rows]:
  // the other 64 N elements are a box's rows further (leading offset; unused with one half),
  // the next 8 tokens follow (stride offset), behind the other half if a box holds only 8.
  const uint32_t lead = (uint32_t)box * 128, stride = box == 8 ? halves * lead : 1024u;
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lead >> 4) << 16) |
         ((uint64_t)(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// The issuer's warp runs its loop as one and one elected lane (`el`) issues.  (With the loop in a
// branch of one lane each product took some 20 cycles longer to issue.)
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc, uint32_t el) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u), "r"(el)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc, uint32_t el) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %6, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u), "r"(el)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar, uint32_t el) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(el)
      : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// Loads are asynchronous: the registers hold the values behind wait_ld(), and the compiler may
// use them only behind this, which ties their uses to the wait.
__device__ __forceinline__ void landed(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void landed(uint32_t (&r)[16]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// 32 columns of this warp's 32 lanes; the registers are valid after wait_ld().
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

// 2^x by the hardware (2 ulp, results below 2^-126 flushed).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations at once (register pairs).
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float block_max(const uint32_t (&v)[2][32]) {
  float a = __uint_as_float(v[0][0]), b = __uint_as_float(v[1][0]);
#pragma unroll
  for (int e = 1; e < 31; e += 2) {
    a = fmaxf(a, fmaxf(__uint_as_float(v[0][e]), __uint_as_float(v[0][e + 1])));
    b = fmaxf(b, fmaxf(__uint_as_float(v[1][e]), __uint_as_float(v[1][e + 1])));
  }
  return fmaxf(fmaxf(a, b), fmaxf(__uint_as_float(v[0][31]), __uint_as_float(v[1][31])));
}

template <int D>
struct Smem {
  static constexpr int kTile = kChunk * 128;              // 128 rows of 128 bytes
  static constexpr int kHalves = D / 64;
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kOperand = kHalves * kTile;        // a Q tile, a K or V chunk
  static constexpr int kQ = 0;                            // 2 Q tiles
  static constexpr int kK = 2 * kOperand;
  static constexpr int kV = kK + kStages * kOperand;
  static constexpr int kBars = kV + kStages * kOperand;
  static constexpr int kNumBars = 4 * kStages + 10 + 2 * kRing;
  static constexpr int kMisc = kBars + 8 * kNumBars;      // tmem slot, abort flag, totals
  static constexpr int kSegs = kMisc + 32;                // [kRing] segments
  static constexpr int kTables = kSegs + 48 * kRing;
};

// Tables of the groups and sequences, in shared or global memory.
struct Tables {
  int* lo;       // [G + 1] first sequence
  int* s;        // [G] shared tokens
  int* leader;   // [G] sequence whose table row is read
  int* rows;     // [G] query rows per KV head
  int* start;    // [G] where its units begin on the scale of costs
  int* unit;     // [G] first unit
  int* len;      // [B] length
  int* gid;      // [B] group or -1
  int* own;      // [B] where its own units begin, behind all shared ones
  __host__ __device__ static size_t ints(int G, int B) { return 6 * (size_t)G + 1 + 3 * (size_t)B; }
  __device__ __forceinline__ void place(int* base, int G, int B) {
    lo = base; s = lo + G + 1; leader = s + G; rows = leader + G; start = rows + G;
    unit = start + G; len = unit + G; gid = len + B; own = gid + B;
  }
};

// First token of a sequence's chunk grid: whole boxes of a page.
__device__ __forceinline__ int own_base(const Params& p, int s) {
  return s & ~(min(p.P, kChunk) - 1);   // a power of two
}
__device__ __forceinline__ int own_chunks(const Params& p, int s, int len) {
  return len > s ? (len - own_base(p, s) + kChunk - 1) / kChunk : 0;
}

// Builds the tables with threads tid = 0 .. nt - 1 (whole warps; barrier 1).  totals: cost of
// the shared units, of all, rows of a tile, chunks in all.  Inlined, so that tables in shared
// memory are accessed as such.
__device__ __forceinline__ void bar1(int nt) { asm volatile("bar.sync 1, %0;" ::"r"(nt) : "memory"); }
__device__ __forceinline__ void build_tables(const TcParams& tp, const Tables& t, int* totals,
                                             int ctas, int tid, int nt) {
  const Params& p = tp.p;
  const int lane = tid & 31;
  // The last warps fetch the groups, the others the lengths: one round trip for both.
#pragma unroll 1
  for (int g = nt - 1 - tid; g <= p.G; g += nt) {
    t.lo[g] = p.G ? p.starts[g] : 0;
    if (g < p.G) {
      t.s[g] = 0x7fffffff;
      t.leader[g] = 0x7fffffff;
      t.unit[g] = p.shared[g];
    }
  }
#pragma unroll 1
  for (int b = tid; b < p.B; b += nt) t.len[b] = seq_len(p, b, true);
  bar1(nt);
#pragma unroll 1
  for (int b = tid; b < p.B; b += nt) {
    const int n = t.len[b];
    int gid = -1;
    if (p.G) {
      int a = 0, z = p.G;     // the last group that starts at or before b
#pragma unroll 1
      while (z - a > 1) {
        const int mid = (a + z) >> 1;
        if (t.lo[mid] <= b) a = mid; else z = mid;
      }
      const int lo = t.lo[a], hi = t.lo[a + 1];
      if (n > 0 && lo >= 0 && hi <= p.B && b >= lo && b < hi && b - lo < p.max_group) {
        gid = a;
        atomicMin(&t.s[a], n);
        atomicMin(&t.leader[a], b);
      }
    }
    t.gid[b] = gid;
  }
  bar1(nt);
  if (tid < 32) {   // the groups, with prefix sums for narrow and for wide tiles
    // One bad range and nothing is shared: overlapping groups would pass the workspace.
    int bad = 0;
#pragma unroll 1
    for (int g = lane; g < p.G; g += 32)
      bad |= t.lo[g] < 0 || t.lo[g + 1] < t.lo[g] || t.lo[g + 1] > p.B;
    bad = __any_sync(0xffffffffu, bad);
    if (bad && lane == 0) atomicOr(p.status, kStatusBadGroup);
    const int narrow = tp.nb * p.R;
    const int per = (p.G + 31) >> 5, g0 = min(lane * per, p.G), g1 = min(g0 + per, p.G);
    int most = 0;
#pragma unroll 1
    for (int g = g0; g < g1; ++g) {   // a lane's groups
      int n = 0, rows = 0;
      if (!bad && t.leader[g] != 0x7fffffff) {
        n = max(0, min(t.unit[g], t.s[g]));
        rows = min(t.lo[g + 1] - t.lo[g], p.max_group) * p.R;
      }
      t.s[g] = n;
      t.rows[g] = rows;
      if (n) most = max(most, rows);
    }
    const bool wide = __reduce_max_sync(0xffffffffu, most) > narrow;
    const int rt = wide ? 2 * narrow : narrow;
    int chunks = 0, units = 0;
#pragma unroll 1
    for (int g = g0; g < g1; ++g) {
      const int u = t.s[g] ? quot(t.rows[g] + rt - 1, rt) * p.Hkv : 0;
      units += u;
      chunks += u * ((t.s[g] + kChunk - 1) >> 7);
    }
    // own chunks and units of this lane's sequences
    const int bper = (p.B + 31) >> 5, b0 = min(lane * bper, p.B), b1 = min(b0 + bper, p.B);
    __syncwarp();
    int oc = 0, ou = 0;
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      int gid = t.gid[b];
      if (gid >= 0 && t.s[gid] == 0) t.gid[b] = gid = -1;
      const int n = own_chunks(p, gid >= 0 ? t.s[gid] : 0, t.len[b]);
      oc += n * p.Hkv;
      ou += n ? p.Hkv : 0;
    }
    const int all = __reduce_add_sync(0xffffffffu, chunks + oc);
    Costs cost;
    cost.set(all, narrow, ctas);
    const Cost own = cost.own();
    int wl = 0;
#pragma unroll 1
    for (int g = g0; g < g1; ++g)
      if (t.s[g])
        wl += quot(t.rows[g] + rt - 1, rt) * p.Hkv *
              cost.shared(t.rows[g]).size((t.s[g] + kChunk - 1) >> 7);
    const int xl = oc * own.chunk + ou * own.unit;
    int cs = wl, us = units, xs = xl;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, cs, o), b = __shfl_up_sync(0xffffffffu, us, o);
      const int d = __shfl_up_sync(0xffffffffu, xs, o);
      if (lane >= o) {
        cs += a;
        us += b;
        xs += d;
      }
    }
    if (lane == 31) {
      totals[0] = cs;
      totals[1] = cs + xs;
      totals[2] = rt;
      totals[3] = all;
    }
    cs -= wl;
    us -= units;
    xs -= xl;
#pragma unroll 1
    for (int g = g0; g < g1; ++g) {
      t.start[g] = cs;
      t.unit[g] = us;
      if (t.s[g]) {
        const int ta = quot(t.rows[g] + rt - 1, rt) * p.Hkv;
        us += ta;
        cs += ta * cost.shared(t.rows[g]).size((t.s[g] + kChunk - 1) >> 7);
      }
    }
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      t.own[b] = xs;
      const int gid = t.gid[b], n = own_chunks(p, gid >= 0 ? t.s[gid] : 0, t.len[b]);
      xs += own.size(n) * p.Hkv;
    }
  }
  bar1(nt);
}

// The plan's entries first, first + step, ...
__device__ __noinline__ void write_plan(const TcParams& tp, const Tables& t, const int* totals,
                                           int ctas, int first, int step) {
  const Params& p = tp.p;
  const int narrow = tp.nb * p.R, rt = totals[2];
  Split split;
  split.set(totals[1], ctas);
  Costs cost;
  cost.set(totals[3], narrow, ctas);
#pragma unroll 1
  for (int e = first; e < p.B * p.Hkv; e += step) {
    const int b = quot(e, p.Hkv), hk = e - b * p.Hkv, g = t.gid[b];
    int4 v = make_int4(0, 0, 0, 0);
    int s = 0;
    if (g >= 0) {
      s = t.s[g];
      const int nch = (s + kChunk - 1) / kChunk, tiles = quot(t.rows[g] + rt - 1, rt);
      const int rr = (b - t.lo[g]) * p.R, tile = quot(rr, rt), u = hk * tiles + tile;
      const bool wide = min(rt, t.rows[g] - tile * rt) > narrow;
      const int q = wide && rr - tile * rt >= narrow ? 1 : 0;
      const Cost c = cost.shared(t.rows[g]);
      const int x = t.start[g] + u * c.size(nch), a = split.owner(x);
      const int segs = split.owner(x + (nch - 1) * c.chunk) - a + 1;
      v.x = 2 * (t.unit[g] + u + a) + q;
      v.z = (wide ? segs : 2 * segs) | (rr - tile * rt - q * narrow) << 16 |
            (wide ? (int)0x80000000 : 0);
    }
    const int nch = own_chunks(p, s, t.len[b]);
    if (nch) {
      const Cost c = cost.own();
      const int x = totals[0] + t.own[b] + hk * c.size(nch), a = split.owner(x);
      v.y = 2 * (e + a);
      v.w = 2 * (split.owner(x + (nch - 1) * c.chunk) - a + 1);
    }
    tp.plan[e] = v;
  }
}

// For batches whose tables do not fit shared memory: one block builds them in global memory.
__global__ void __launch_bounds__(1024) tables_kernel(const __grid_constant__ TcParams tp) {
  __shared__ int totals[4];
  pdl_wait();
  Tables t;
  t.place(tp.tables, tp.p.G, tp.p.B);
  build_tables(tp, t, totals, tp.ctas, threadIdx.x, blockDim.x);
  __syncthreads();
  if (threadIdx.x < 4) tp.heads[threadIdx.x] = totals[threadIdx.x];
  pdl_launch_dependents();
}

// A segment: the part of a unit in a CTA's range.  The producer walks them and publishes
// each in a ring in shared memory; n = 0 ends the list.
struct __align__(16) Segment {
  int n;         // chunks
  int wide;
  int t0;        // first token of the segment's first chunk
  int hi;        // end of the unit's tokens
  int lo;        // their start
  int rows, slot, own;   // slot: first of its two
  int hk, b_table, b_q, pad;
};
static_assert(sizeof(Segment) == 48, "ring entries of 48 bytes");

// Walks the segments of the chunks that begin in [x, x1).
struct Walker {
  int x, x1, g, b, X0, rt;   // X0: cost of the shared units
  Costs cost;

  // The last of n ascending entries that is <= x (0 if none), by a whole warp.
  static __device__ __noinline__ int find(const int* a, int n, int x) {
    const int lane = threadIdx.x & 31;
    int lo = 0;
#pragma unroll 1
    while (n > 1) {
      const int step = (n + 31) >> 5, i = lane * step;
      const int k = __popc(__ballot_sync(0xffffffffu, i < n && a[lo + i] <= x));
      const int at = k ? (k - 1) * step : 0;
      lo += at;
      n = min(step, n - at);
    }
    return lo;
  }
  __device__ __forceinline__ void init(const TcParams& tp, const Tables& t, const int* totals) {
    const Params& p = tp.p;
    X0 = totals[0];
    rt = totals[2];
    cost.set(totals[3], tp.nb * p.R, gridDim.x);
    Split split;
    split.set(totals[1], gridDim.x);
    const bool idle = (int)blockIdx.x >= split.C;
    x = idle ? 0 : split.start(blockIdx.x);
    x1 = idle ? 0 : split.start(blockIdx.x + 1);
    g = x < X0 ? find(t.start, p.G, x) : 0;
    b = x1 > X0 ? find(t.own, p.B, max(0, x - X0)) : 0;
  }
  __device__ __forceinline__ bool next(const TcParams& tp, const Tables& t, Segment& sg) {
    const Params& p = tp.p;
#pragma unroll 1
    while (x < x1) {
      int j0, j1;
      if (x < X0) {
        int nch, tiles, size;
        Cost c;
#pragma unroll 1
        while (true) {   // the group that holds x
          nch = (t.s[g] + kChunk - 1) / kChunk;
          tiles = quot(t.rows[g] + rt - 1, rt);
          c = cost.shared(t.rows[g]);
          size = c.size(nch);
          if (x < t.start[g] + size * tiles * p.Hkv || g + 1 >= p.G) break;
          ++g;
        }
        const int y = x - t.start[g], ul = quot(y, size), base = x - (y - ul * size);
        j0 = c.chunk_from(x - base);
        j1 = min(nch, c.chunk_from(x1 - base));
        x = min(x1, base + size);
        sg.hk = quot(ul, tiles);
        const int tile = ul - sg.hk * tiles;
        sg.own = 0;
        sg.b_table = t.leader[g];
        sg.b_q = t.lo[g] + tile * (rt > tp.nb * p.R ? 2 * tp.nb : tp.nb);
        sg.rows = min(rt, t.rows[g] - tile * rt);
        sg.wide = sg.rows > tp.nb * p.R;
        sg.t0 = j0 * kChunk;
        sg.lo = 0;
        sg.hi = t.s[g];
        sg.slot = 2 * (t.unit[g] + ul + (int)blockIdx.x);
      } else {
        const Cost c = cost.own();
        int nch, s, size;
#pragma unroll 1
        while (true) {   // the sequence that holds x
          s = t.gid[b] >= 0 ? t.s[t.gid[b]] : 0;
          nch = own_chunks(p, s, t.len[b]);
          size = c.size(nch);
          if (x - X0 < t.own[b] + size * p.Hkv || b + 1 >= p.B) break;
          ++b;
        }
        const int y = x - X0 - t.own[b], hk = quot(y, size), base = x - (y - hk * size);
        j0 = c.chunk_from(x - base);
        j1 = min(nch, c.chunk_from(x1 - base));
        x = min(x1, base + size);
        sg.own = 1;
        sg.hk = hk;
        sg.b_table = b;
        sg.b_q = b;
        sg.rows = p.R;
        sg.wide = 0;
        sg.t0 = own_base(p, s) + j0 * kChunk;
        sg.lo = s;
        sg.hi = t.len[b];
        sg.slot = 2 * (b * p.Hkv + hk + (int)blockIdx.x);
      }
      sg.n = j1 - j0;
      if (sg.n > 0) return true;   // none: x was in the last chunk of its unit
    }
    return false;
  }
};

// The issuer's place in the items of the CTA.
struct Cursor {
  int n, wide, t0, hi;             // of the segment; n = 0: past the last
  int j, sub, item, k, qc, seg;    // chunk and row tile in the segment; running counters
};

template <int D, typename T, bool kGlobalTables>
__global__ void __launch_bounds__(kThreads, 1)
parts_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
             const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_q1,
             const __grid_constant__ TcParams tp) {
  using S = Smem<D>;
  constexpr int NS = S::kStages;
  constexpr uint32_t FMT = __is_same(T, __nv_bfloat16) ? 1u : 0u;
  // fp32 accumulate, M = 128; S: both K-major, N = tokens; P V: N = D, V MN-major (bit 16).
  constexpr uint32_t ID_S = (1u << 4) | (FMT << 7) | (FMT << 10) | (8u << 24);
  constexpr uint32_t ID_O = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) |
                            ((uint32_t)(D >> 3) << 17) | (8u << 24);
  const Params& p = tp.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sb = smem_u32(smem);
  const uint32_t bars = sb + S::kBars;
  const uint32_t kfull = bars, kempty = kfull + 8 * NS, vfull = kempty + 8 * NS,
                 vempty = vfull + 8 * NS, sfull = vempty + 8 * NS, pready = sfull + 16,
                 ofull = pready + 16, qfull = ofull + 16, qempty = qfull + 16,
                 gfull = qempty + 16, gempty = gfull + 8 * kRing;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kMisc + 4);
  int* totals = reinterpret_cast<int*>(smem + S::kMisc + 8);
  const Segment* segs = reinterpret_cast<const Segment*>(smem + S::kSegs);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(kfull + 8 * i, 1);
      mbar_init(kempty + 8 * i, 1);
      mbar_init(vfull + 8 * i, 1);
      mbar_init(vempty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sfull + 8 * i, 1);
      mbar_init(pready + 8 * i, 128);
      mbar_init(ofull + 8 * i, 1);
      mbar_init(qfull + 8 * i, 1);
      mbar_init(qempty + 8 * i, 1);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(gfull + 8 * i, 1);
      mbar_init(gempty + 8 * i, 10);   // the issuer, the V producer, eight softmax warps
    }
    *abort_flag = 0;
    fence_mbarrier_init();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_q1);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_launch_dependents();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  Tables t;
  if (kGlobalTables)
    t.place(tp.tables, p.G, p.B);
  else
    t.place(reinterpret_cast<int*>(smem + S::kTables), p.G, p.B);

  // Registers: 12 warps, three per scheduler, start with 168 each (504 of a scheduler's 512 a
  // lane); the softmax warps take what the others give up.
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  pdl_wait();               // lengths, queries and pages come from earlier kernels
  if (kGlobalTables) {      // built by tables_kernel
    if (tid < 256 + 4) totals[tid - 256] = tp.heads[tid - 256];
    bar1(128);
  } else {
    build_tables(tp, t, totals, gridDim.x, tid - 256, 128);
  }
  if (warp == 8 || warp == 10) {
    // ---- TMA producers: lane i brings page (or part of a page) i of the chunk.  Warp 8
    // walks the segments, publishes them and brings Q and K, warp 10 brings V. ----
    const bool isv = warp == 10;
    const int box = min(p.P, kChunk), bsh = 31 - __clz(box);   // box rows: a power of two
    const int ppc = kChunk >> bsh;                             // boxes per chunk
    const uint32_t tile0 = sb + (isv ? S::kV : S::kK);
    const uint32_t fulls = isv ? vfull : kfull, empties = isv ? vempty : kempty;
    int k = 0, qc = 0;
    Walker w0;
    if (!isv) w0.init(tp, t, totals);
#pragma unroll 1
    for (int ns = 0;; ++ns) {
      Segment sg;
      const int slot = ns % kRing;
      Segment* entry = reinterpret_cast<Segment*>(smem + S::kSegs) + slot;
      if (!isv) {
        if (!w0.next(tp, t, sg)) sg.n = 0;
        wait(gempty + 8 * slot, ((ns / kRing) & 1) ^ 1, abort_flag, p.status);
        if (lane == 0) {
          *entry = sg;
          mbar_arrive(gfull + 8 * slot);
        }
        __syncwarp();
      } else {
        wait(gfull + 8 * slot, (ns / kRing) & 1, abort_flag, p.status);
        sg = *entry;
        __syncwarp();
        if (lane == 0) mbar_arrive(gempty + 8 * slot);
      }
      if (__any_sync(0xffffffffu, sg.n == 0 || *abort_flag != 0)) break;
      const int32_t* row = p.block_table + (long long)sg.b_table * p.max_pages;
      auto page_at = [&](int j) -> int {
        const int tok = sg.t0 + j * kChunk + (lane << bsh);
        if (j >= sg.n || lane >= ppc || tok >= sg.hi) return 0;
        return row[p.P <= kChunk ? tok >> bsh : quot(tok, p.P)];
      };
      int next = page_at(0);
      if (!isv) {
#pragma unroll 1
        for (int q = 0; q <= sg.wide; ++q, ++qc) {
          const int qb = qc & 1;
          wait(qempty + 8 * qb, ((qc >> 1) & 1) ^ 1, abort_flag, p.status);
          if (lane == 0 && !*abort_flag) {
            mbar_arrive_expect_tx(qfull + 8 * qb, (uint32_t)((sg.own ? 1 : tp.nb) * p.R * D * 2));
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
              tma_load_3d(sb + S::kQ + qb * S::kOperand + h * S::kTile, sg.own ? &map_q1 : &map_q,
                          h * 64, sg.hk * p.R, sg.b_q + q * tp.nb, qfull + 8 * qb);
          }
          __syncwarp();
        }
      }
#pragma unroll 1
      for (int j = 0; j < sg.n; ++j, ++k) {
        const int st = k % NS;
        const int t0 = sg.t0 + j * kChunk;
        const int boxes = min(ppc, (sg.hi - t0 + box - 1) >> bsh);
        int page = next;
        next = page_at(j + 1);
        if (page < 0 || page >= p.num_pages) {
          atomicOr(p.status, kStatusBadPage);
          page = 0;
        }
        int in_page = 0;      // a page of more than a chunk: where in it
        if (p.P > kChunk) in_page = t0 - quot(t0, p.P) * p.P;
        const int y = (page * p.Hkv + sg.hk) * p.P + in_page;   // pool rows: below 2^31
        wait(empties + 8 * st, ((k / NS) & 1) ^ 1, abort_flag, p.status);
        const bool go = !*abort_flag;
        const uint32_t full = fulls + 8 * st;
        if (lane == 0 && go) mbar_arrive_expect_tx(full, (uint32_t)(boxes * box * D * 2));
        __syncwarp();
        if (go && lane < boxes) {
          const uint32_t dst = tile0 + st * S::kOperand;
          if (isv) {       // [box][half][rows]: both halves in one copy
            tma_load_3d(dst + lane * (box * 128 * S::kHalves), &map_v, 0, y, 0, full);
          } else {         // [half][rows of all boxes]: 8-row groups evenly spaced
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
              tma_load_2d(dst + lane * box * 128 + h * S::kTile, &map_k, h * 64, y, full);
          }
        }
        __syncwarp();
      }
    }
    if (*abort_flag) {   // let the copies in flight land before the block goes
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {
      }
    }
  } else if (warp == 11) {
    write_plan(tp, t, totals, gridDim.x, blockIdx.x * 32 + lane, gridDim.x * 32);
  } else if (warp == 9) {
    // ---- tcgen05 issuer ----
    asm volatile("bar.sync 2, 288;" ::: "memory");   // the softmax warps' rehearsal is over
    const uint32_t el = elect_one();
    // Segment entries are read once by each cursor; b's read gives the entry back.
    auto load = [&](Cursor& c, bool last) {
      const int slot = c.seg % kRing;
      wait(gfull + 8 * slot, (c.seg / kRing) & 1, abort_flag, p.status);
      const int4 v = *reinterpret_cast<const int4*>(smem + S::kSegs + 48 * slot);
      c.n = *abort_flag ? 0 : v.x;
      c.wide = v.y; c.t0 = v.z; c.hi = v.w;
      c.j = 0;
      __syncwarp();
      if (last && el) mbar_arrive(gempty + 8 * slot);
      ++c.seg;
    };
    auto advance = [&](Cursor& c, bool last) {
      ++c.item;
      if (c.wide && c.sub == 0) {
        c.sub = 1;
        return;
      }
      c.sub = 0;
      ++c.k;
      if (++c.j == c.n) {
        c.qc += 1 + c.wide;
        load(c, last);
      }
    };
    auto tokens = [](const Cursor& c) { return min(kChunk, c.hi - c.t0 - c.j * kChunk); };
    // V: 16 tokens of a k-step are inside a box, or two boxes of 8 (descriptor units of 16 B)
    const int vbox = min(p.P, kChunk), vsh = 31 - __clz(vbox), vstep = vbox * 8 * S::kHalves;
    Cursor a = {}, b = {};     // S (a) runs two items ahead of P V (b)
    load(a, false);
    load(b, true);
    uint32_t ready = 0;        // bit s: parity of stream s's next P
#pragma unroll 1
    for (int lead = 2; b.n;) {
      if (lead) {
        --lead;
      } else {                 // O += P V
        const int s = b.item & 1, st = b.k % NS;
        wait(pready + 8 * s, (ready >> s) & 1, abort_flag, p.status);
        if (b.sub == 0) wait(vfull + 8 * st, (b.k / NS) & 1, abort_flag, p.status);
        fence_after();
        const uint64_t vd = desc_mnmajor(sb + S::kV + st * S::kOperand, vbox, S::kHalves);
        const bool first = b.wide ? b.j == 0 : b.j < 2;
        const int steps = (tokens(b) + 15) >> 4;
#pragma unroll
        for (int kk = 0; kk < kChunk / 16; ++kk) {
          if (kk >= steps) continue;
          mma_ts(tmem + 256 + s * D, tmem + s * 128 + kk * 8,
                 vd + (((kk * 16) >> vsh) * vstep + ((kk * 16) & (vbox - 1)) * 8), ID_O,
                 !first || kk > 0, el);
        }
        ready ^= 1u << s;
        if (!b.wide || b.sub == 1) commit(vempty + 8 * st, el);
        if (b.wide ? b.j == b.n - 1 : b.j >= b.n - 2) commit(ofull + 8 * s, el);
        advance(b, true);
      }
      if (a.n) {               // S = Q K^T
        const int s = a.item & 1, st = a.k % NS, qi = a.qc + a.sub, qb = qi & 1;
        if (a.j == 0) wait(qfull + 8 * qb, (qi >> 1) & 1, abort_flag, p.status);
        if (a.sub == 0) wait(kfull + 8 * st, (a.k / NS) & 1, abort_flag, p.status);
        fence_after();
        const uint64_t qd = desc_kmajor(sb + S::kQ + qb * S::kOperand);
        const uint64_t kd = desc_kmajor(sb + S::kK + st * S::kOperand);
        const uint32_t id = ID_S | ((uint32_t)((tokens(a) + 31) >> 5 << 2) << 17);   // N = 32, 64 ...
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = ((kk / 4) * S::kTile + (kk % 4) * 32) >> 4;
          mma_ss(tmem + s * 128, qd + off, kd + off, id, kk > 0, el);
        }
        commit(sfull + 8 * s, el);
        if (!a.wide || a.sub == 1) commit(kempty + 8 * st, el);
        if (a.j == a.n - 1) commit(qempty + 8 * qb, el);
        advance(a, false);
      }
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax: thread = query row ----
    // The first round is a rehearsal on whatever TMEM holds, before any S is issued, while
    // the tables are built: it brings the code into the instruction caches.  A decode step
    // streams its weights between two launches, so they are cold (measured: 18 thousand
    // cycles for the first item without it).
    const int s = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + s * 128, to = tmem + lanes + 256 + s * D;
    const float kNegInf = __int_as_float(0xff800000);
    const float sc = p.scale_log2;                     // positive
    const uint64_t sc2 = pair(sc, sc);
    // the scaled score whose weight is 1
    auto zero_of = [&](float m) { return m == kNegInf ? 0.f : fmaf(m, sc, -kScale<T>); };
    const int narrow = tp.nb * p.R;
    const int box = min(p.P, kChunk), bsh = 31 - __clz(box);
    int k = 0, it = 0, n_items = 0, n_o = 0;
    Segment sg;
    sg.n = 2; sg.wide = 0; sg.t0 = 0; sg.hi = 2 * kChunk - 1; sg.lo = 0; sg.rows = 128; sg.slot = 0;
    sg.own = 0;
#pragma unroll 1
    for (int ns = -1;; ++ns) {
      const bool real = ns >= 0;
      if (real) {
        const int slot = ns % kRing;
        wait(gfull + 8 * slot, (ns / kRing) & 1, abort_flag, p.status);
        const int4* e = reinterpret_cast<const int4*>(segs + slot);
        const int4 x = e[0], y = e[1];
        sg.n = x.x; sg.wide = x.y; sg.t0 = x.z; sg.hi = x.w;
        sg.lo = y.x; sg.rows = y.y; sg.slot = y.z; sg.own = y.w;
        __syncwarp();
        if (lane == 0) mbar_arrive(gempty + 8 * slot);
        // after a wait that gave up the entry means nothing; a warp leaves as one
        if (__any_sync(0xffffffffu, sg.n == 0 || *abort_flag != 0)) break;
      }
      // q: row tile of this stream (wide), or whether it has the even or the odd chunks.
      const int q = s ^ (it & 1);
      const int first = sg.wide ? 0 : q, step = sg.wide ? 1 : 2;
      const int rows = sg.wide ? min(narrow, sg.rows - q * narrow) : sg.rows;
      const bool warp_on = (warp & 3) * 32 < rows;
      float m = kNegInf;
      uint64_t l2 = pair(0.f, 0.f);
#pragma unroll 1
      for (int j = first; j < sg.n; j += step) {
        const int t0 = sg.t0 + j * kChunk;
        const int hi = min(kChunk, sg.hi - t0), lo = max(0, sg.lo - t0);
        const int nb = (hi + 31) >> 5;
        if (real) wait(sfull + 8 * s, n_items & 1, abort_flag, p.status);
        fence_after();
        if (warp_on) {
          // Tokens outside the unit: -inf in TMEM, in the few blocks that have any.
          if (lo > 0 || hi < kChunk) {
#pragma unroll 1
            for (int x = 0; x < ((hi + 63) & ~63); x += 16) {
              if (x >= lo && x + 16 <= hi) continue;
              uint32_t o[16];
              if (x < hi && x + 16 > lo) {
                ld16(ts + x, o);
                wait_ld();
                landed(o);
              }
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (x + e < lo || x + e >= hi) o[e] = __float_as_uint(kNegInf);
              st16(ts + x, o);
            }
            wait_st();
          }
          const bool start = j == first, two = nb > 2;
          uint32_t v0[2][32], v1[2][32], w[2][16];
          ld32(ts, v0[0]);
          ld32(ts + 32, v0[1]);
          if (two) {
            ld32(ts + 64, v1[0]);
            ld32(ts + 96, v1[1]);
          }
          wait_ld();
          landed(v0[0]);
          landed(v0[1]);
          float mx = block_max(v0);
          if (two) {
            landed(v1[0]);
            landed(v1[1]);
            mx = fmaxf(mx, block_max(v1));
          }
          // Raise the reference maximum where the weights would grow too large.
          const bool raise = start || (mx - m) * sc > kLag<T>;
          if (__any_sync(0xffffffffu, raise)) {
            const float f = !raise ? 1.f : m == kNegInf ? 0.f : ex2((m - mx) * sc);
            m = raise ? mx : m;
            float a, b;
            unpair(l2, a, b);
            l2 = pair(a * f, b * f);
            if (!start) {
#pragma unroll 1
              for (int y = 0; y < D; y += 16) {
                uint32_t o[16];
                ld16(to + y, o);
                wait_ld();
                landed(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                st16(to + y, o);
              }
            }
          }
          const float ms = zero_of(m);
          const uint64_t nm2 = pair(-ms, -ms);
          auto weigh = [&](const uint32_t (&v)[2][32]) {
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              float a, b;
              unpair(fma2(pair(__uint_as_float(v[e / 32][e % 32]),
                               __uint_as_float(v[e / 32][e % 32 + 1])), sc2, nm2), a, b);
              a = ex2(a);
              b = ex2(b);
              l2 = add2(l2, pair(a, b));
              w[e / 32][e % 32 / 2] = Mma<T>::pack(a, b);
            }
          };
          weigh(v0);               // P's columns lie over S columns that have been read
          st16(ts, w[0]);
          st16(ts + 16, w[1]);
          if (two) {
            weigh(v1);
            st16(ts + 32, w[0]);
            st16(ts + 48, w[1]);
          }
          wait_st();
        }
        if (real) {
          const int end = (hi + 15) & ~15;     // of P V's last step
          if (hi < end && (!sg.wide || q == 0)) {
            // Rows of V behind the last token hold anything; a weight 0 would not silence a
            // NaN.  S of this item follows the products of the stream's item before, so the
            // stage's earlier chunk is done: this wait cannot take its phase for the chunk's.
            const int st = (k + j) % NS;
            wait(vfull + 8 * st, ((k + j) / NS) & 1, abort_flag, p.status);
            const uint32_t v0 = sb + S::kV + st * S::kOperand;
            const int per = (end - hi) * 8;
#pragma unroll 1
            for (int i = r; i < per * S::kHalves; i += 128) {
              const int h = i >= per ? 1 : 0, w = i - h * per, tok = hi + (w >> 3);
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                               v0 + (tok >> bsh) * (box * 128 * S::kHalves) + h * (box * 128) +
                               (tok & (box - 1)) * 128 + (w & 7) * 16),
                           "r"(0u)
                           : "memory");
            }
            fence_proxy_async_smem();
          }
          fence_before();
          mbar_arrive(pready + 8 * s);
          ++n_items;
        }
      }
      // ---- segment end: this stream's partial ----
      const long long slot = sg.slot + q;
      const int rs = sg.own ? p.R : tp.rs;
      float4* po = reinterpret_cast<float4*>(sg.own ? tp.own_o : p.part_o) + slot * rs * (D / 4);
      float* pl = (sg.own ? tp.own_lse : p.part_lse) + slot * rs;
      const bool write = real && r < rows;
      if (first < sg.n) {
        if (real) {
          wait(ofull + 8 * s, n_o & 1, abort_flag, p.status);
          ++n_o;
        }
        fence_after();
        if (warp_on) {
          float a, b;
          unpair(l2, a, b);
          const float l = a + b;
          const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
          for (int x = 0; x < D / 32; ++x) {
            uint32_t o[32];
            ld32(to + 32 * x, o);
            wait_ld();
            landed(o);
            if (write) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                po[(8 * x + e / 4) * rs + r] = make_float4(
                    __uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv,
                    __uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
            }
          }
          if (write) pl[r] = l == 0.f ? kNegInf : zero_of(m) + log2f(l);
        }
        fence_before();   // O is read: the next segment's products may overwrite it
      } else if (write) {
        pl[r] = kNegInf;  // a single chunk, on the other stream
      }
      if (real) {
        k += sg.n;
        it += sg.wide ? 2 * sg.n : sg.n;
      } else {
        pdl_wait();       // what follows overwrites partials that the last join may still read
        fence_before();
        asm volatile("bar.sync 2, 288;" ::: "memory");
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 9)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u)
                 : "memory");
}

// ---------------------------------------------------------------------------------
// join_kernel: D / 4 lanes per output row, each with 4 of its elements.  The lanes first
// share the parts' log2-sum-exps (a part each), then all run over the parts.
template <int D, typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ TcParams tp) {
  constexpr int LPR = D / 4;
  const Params& p = tp.p;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & (LPR - 1);
  const long long row = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const unsigned mask = LPR == 32 ? 0xffffffffu
                                  : 0xffffu << (threadIdx.x & 16);
  if (row >= (long long)p.B * p.Hq) return;
  const int hkr = quot((int)row, p.R), rh = (int)row - hkr * p.R;   // (b, KV head), head
  const int4 v = tp.plan[hkr];
  const float kNegInf = __int_as_float(0xff800000);
  float M = kNegInf, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  // The parts of a unit: slots first, first + 1, ... or every second of them.
  auto add = [&](const float* lse, const float4* o, int rs, int parts, int step) {
    for (int e0 = 0; e0 < parts; e0 += LPR) {
      const int n = min(LPR, parts - e0);
      const float mine = lane < n ? lse[(long long)(e0 + lane) * step * rs] : kNegInf;
      float top = mine;
#pragma unroll
      for (int x = LPR / 2; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, x, LPR));
      const float nm = fmaxf(M, top);
      const float mu = nm == kNegInf ? 0.f : nm;
      const float f = ex2(M - mu);
      M = nm;
      L *= f;
      acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
      const float wm = ex2(mine - mu);
      const float4* src = o + (long long)e0 * step * rs * (D / 4);
      for (int e1 = 0; e1 < n; e1 += 8) {   // eight parts' loads in flight
        float4 x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e1 + e < n) x[e] = src[(long long)(e1 + e) * step * rs * (D / 4)];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = __shfl_sync(mask, wm, (e1 + e) & (LPR - 1), LPR);
          if (e1 + e >= n || w == 0.f) continue;   // an empty part's O is not written
          L += w;
          acc.x = fmaf(x[e].x, w, acc.x); acc.y = fmaf(x[e].y, w, acc.y);
          acc.z = fmaf(x[e].z, w, acc.z); acc.w = fmaf(x[e].w, w, acc.w);
        }
      }
    }
  };
  if (v.z) {
    const long long slot = v.x;
    const int tr = ((v.z >> 16) & 0x7fff) + rh;
    add(p.part_lse + slot * tp.rs + tr,
        reinterpret_cast<const float4*>(p.part_o) + (slot * (D / 4) + lane) * tp.rs + tr, tp.rs,
        v.z & 0xffff, v.z < 0 ? 2 : 1);
  }
  if (v.w) {
    const long long slot = v.y;
    add(tp.own_lse + slot * p.R + rh,
        reinterpret_cast<const float4*>(tp.own_o) + (slot * (D / 4) + lane) * p.R + rh, p.R, v.w, 1);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;     // an empty sequence gives zeros
  uint2 r;
  r.x = Mma<T>::pack(acc.x * inv, acc.y * inv);
  r.y = Mma<T>::pack(acc.z * inv, acc.w * inv);
  reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + row * D)[lane] = r;
}

}  // namespace tc
}  // namespace prefix
}  // namespace llmc
