// Shared-prefix decode attention on the tensor cores: bf16/fp16, head size 64 or 128.
//
// Two launches.  prefix_kernel computes the shared parts, own_kernel the sequences' own
// parts and the join; own_kernel's attention needs nothing of prefix_kernel, so under
// programmatic dependent launch it runs beside it and waits only before the join.
//
// prefix_kernel: rows = the query rows of a group that use one KV head (sequence, then
// head), cut into tiles; a (group, KV head, row tile) is a unit, its tokens are cut into
// chunks of 128, the chunks of all units are laid end to end, and CTA c of the persistent
// grid takes chunks [c W / C, (c + 1) W / C) of the W.  The part of a unit inside a CTA's
// range (a segment) leaves one partial in slot unit + c, which is unique because both
// orders ascend.
//   warps 0-3, 4-7   two softmax warpgroups ("streams"), one query row per thread;
//   warp 8           TMA producer: pages of K and V into 128-byte-swizzled tiles;
//   warp 9           tcgen05 issuer: S = Q K^T (both in shared memory), O += P V (P in
//                    TMEM over S's columns, V as an MN-major operand, so no transpose).
// TMEM: S and O of both streams, 4 x 128 fp32 columns at head size 128 = all 512.
// Row tiles of 128: chunks alternate between the streams (each with its own running
// maximum, sum and O, joined through shared memory at the segment's end), so the softmax
// of one chunk runs under the products of the next.  Row tiles of 256: a stream has 128 of
// the rows and every chunk serves both, which halves the K/V traffic per row; used when
// the work is long enough (see kLongChunks).
// The running maximum is only raised when it would grow by more than 8 (log2): weights up
// to 2^8 are harmless in 16 bits, and O is then rarely rescaled.
#pragma once

#include "shared_prefix.cuh"

namespace llmc {
namespace prefix {
namespace tc {

constexpr int kChunk = 128;        // tokens of a chunk (MMA N of S, K of P V)
constexpr int kThreads = 320;
constexpr int kMaxGroups = 1024;   // group tables in shared memory: 24 bytes each

// Row tiles of 256 from this many 256-row chunks per CTA on.
constexpr int kLongChunks = 6;

struct Plan {          // written by prefix_kernel's first CTA, read by own_kernel
  int W, rt, pad[6];   // chunks in all, rows of a tile; then 4 ints per group:
};                     // first chunk, first unit, chunks of a unit, rows

struct TcParams {
  Params p;
  int32_t* plan;
  int rs_a, rs_b;      // rows of a slot with row tiles of 128 / 256
  int ctas;            // grid of prefix_kernel
};

__device__ __forceinline__ int cta_start(int c, int W, int C) {
  return (int)((long long)c * W / C);
}
__device__ __forceinline__ int cta_owner(int u, int W, int C) {
  int c = (int)((long long)u * C / W);
  while (c + 1 < C && cta_start(c + 1, W, C) <= u) ++c;
  while (c > 0 && cta_start(c, W, C) > u) --c;
  return c;
}

// ---- tcgen05 -------------------------------------------------------------------
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t addr) {
  // 128-byte swizzle, rows of 128 bytes: 8-row groups 1024 bytes apart.
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) |
         (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t addr) {
  // 128-byte swizzle, 64 contiguous N elements per row (a token), 8-token groups 1024 bytes
  // apart (stride offset), the next 64 N elements kChunk rows further (leading offset).
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(kChunk * 128 / 16) << 16) |
         (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
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
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
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
__device__ __forceinline__ void bar_softmax() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int D>
struct Smem {
  static constexpr int kTile = kChunk * 128;              // 128 rows of 128 bytes
  static constexpr int kHalves = D / 64;
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kOperand = kHalves * kTile;        // a Q tile, a K or V chunk
  static constexpr int kQ = 0;                            // 2 Q tiles; the join's exchange
  static constexpr int kK = 2 * kOperand;
  static constexpr int kV = kK + kStages * kOperand;
  static constexpr int kBars = kV + kStages * kOperand;
  static constexpr int kNumBars = 4 * kStages + 7;
  static constexpr int kMisc = kBars + 8 * kNumBars;      // tmem slot, abort flag, totals
  static constexpr int kMl = kMisc + 24;                  // [2][128] (max, sum)
  static constexpr int kGroups = kMl + 2 * 128 * 8;
  static size_t bytes(int G) { return 1024 + kGroups + sizeof(int) * (6 * (size_t)G + 1); }
};

// A segment: the part of a unit in this CTA's range.
struct Segment {
  int g, hk, tile, unit, ch0, n, s, leader, lo, rows;   // rows: valid rows of the tile
};

// Group tables in shared memory.
struct Groups {
  int* start;    // [G] first chunk of the group
  int* unit;     // [G] first unit
  int* s;        // [G] shared tokens
  int* leader;   // [G] sequence whose table row is read
  int* lo;       // [G + 1] first sequence
  int* rows;     // [G] query rows per KV head
};

__device__ __forceinline__ bool next_segment(const TcParams& tp, const Groups& gr, int rt, int& c,
                                             int c1, int& g, Segment& sg) {
  if (c >= c1) return false;
  const int G = tp.p.G, Hkv = tp.p.Hkv;
  int nch, tiles;
  while (true) {   // the group that holds chunk c
    nch = (gr.s[g] + kChunk - 1) / kChunk;
    tiles = (gr.rows[g] + rt - 1) / rt;
    if (c < gr.start[g] + nch * tiles * Hkv || g + 1 >= G) break;
    ++g;
  }
  const int x = c - gr.start[g], ul = x / nch;
  sg.g = g;
  sg.hk = ul / tiles;
  sg.tile = ul - sg.hk * tiles;
  sg.unit = gr.unit[g] + ul;
  sg.ch0 = x - ul * nch;
  sg.n = min(nch - sg.ch0, c1 - c);
  sg.s = gr.s[g];
  sg.leader = gr.leader[g];
  sg.lo = gr.lo[g];
  sg.rows = min(rt, gr.rows[g] - sg.tile * rt);
  c += sg.n;
  return true;
}

template <int D, typename T>
__global__ void __launch_bounds__(kThreads, 1)
prefix_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
              const __grid_constant__ TcParams tp) {
  using S = Smem<D>;
  constexpr int NS = S::kStages;
  constexpr uint32_t FMT = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u;
  // fp32 accumulate, M = 128; S: N = 128, both K-major; P V: N = D, V MN-major (bit 16).
  constexpr uint32_t ID_S = (1u << 4) | (FMT << 7) | (FMT << 10) | ((uint32_t)(kChunk >> 3) << 17) |
                            (8u << 24);
  constexpr uint32_t ID_O = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) |
                            ((uint32_t)(D >> 3) << 17) | (8u << 24);
  const Params& p = tp.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sb = smem_u32(smem);
  const uint32_t bars = sb + S::kBars;
  const uint32_t kfull = bars, kempty = kfull + 8 * NS, vfull = kempty + 8 * NS,
                 vempty = vfull + 8 * NS, sfull = vempty + 8 * NS, pready = sfull + 16,
                 ofull = pready + 16, qready = ofull + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kMisc + 4);
  int* total = reinterpret_cast<int*>(smem + S::kMisc + 8);   // W, rt
  float2* ml = reinterpret_cast<float2*>(smem + S::kMl);
  Groups gr;
  gr.start = reinterpret_cast<int*>(smem + S::kGroups);
  gr.unit = gr.start + p.G;
  gr.s = gr.unit + p.G;
  gr.leader = gr.s + p.G;
  gr.rows = gr.leader + p.G;
  gr.lo = gr.rows + p.G;
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
    }
    mbar_init(qready, 256);
    *abort_flag = 0;
    fence_mbarrier_init();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();               // lengths, queries and pages come from earlier kernels
  pdl_launch_dependents();  // after the wait: what own_kernel reads early is then final

  // ---- the groups and this CTA's range ----
  for (int g = tid; g <= p.G; g += kThreads) {
    gr.lo[g] = p.starts[g];
    if (g < p.G) {
      gr.s[g] = 0x7fffffff;
      gr.leader[g] = 0x7fffffff;
    }
  }
  __syncthreads();
  for (int b = tid; b < p.B; b += kThreads) {
    const int n = seq_len(p, b, false);
    if (n <= 0) continue;
    int a = 0, z = p.G;     // the last group that starts at or before b
    while (z - a > 1) {
      const int mid = (a + z) >> 1;
      if (gr.lo[mid] <= b) a = mid; else z = mid;
    }
    const int lo = gr.lo[a], hi = gr.lo[a + 1];
    if (lo >= 0 && hi <= p.B && b >= lo && b < hi && b - lo < p.max_group) {
      atomicMin(&gr.s[a], n);
      atomicMin(&gr.leader[a], b);
    }
  }
  // One bad range and nothing is shared: overlapping groups would pass the workspace.
  int bad = 0;
  for (int g = tid; g < p.G; g += kThreads)
    bad |= gr.lo[g] < 0 || gr.lo[g + 1] < gr.lo[g] || gr.lo[g + 1] > p.B;
  bad = __syncthreads_or(bad);
  if (bad && tid == 0) atomicOr(p.status, kStatusBadGroup);
  for (int g = tid; g < p.G; g += kThreads) {
    const bool any = !bad && gr.leader[g] != 0x7fffffff;
    gr.s[g] = any ? max(0, min(p.shared[g], gr.s[g])) : 0;
    gr.rows[g] = any ? min(gr.lo[g + 1] - gr.lo[g], p.max_group) * p.R : 0;
  }
  __syncthreads();
  if (warp == 0) {
    int rt = 128, w = 0;
    for (int pass = 0; pass < 2; ++pass) {
      // pass 0: would row tiles of 256 give every CTA kLongChunks?  pass 1: the prefix sums
      rt = pass == 0 ? 256 : rt;
      int u = 0, most = 0;
      w = 0;
      for (int g0 = 0; g0 < p.G; g0 += 32) {
        const int g = g0 + lane;
        int units = 0, chunks = 0;
        if (g < p.G && gr.s[g] > 0) {
          units = (gr.rows[g] + rt - 1) / rt * p.Hkv;
          chunks = units * ((gr.s[g] + kChunk - 1) / kChunk);
          most = max(most, gr.rows[g]);
        }
        int cs = chunks, us = units;
        for (int o = 1; o < 32; o <<= 1) {
          const int a = __shfl_up_sync(0xffffffffu, cs, o), b = __shfl_up_sync(0xffffffffu, us, o);
          if (lane >= o) {
            cs += a;
            us += b;
          }
        }
        if (pass == 1 && g < p.G) {
          gr.start[g] = w + cs - chunks;
          gr.unit[g] = u + us - units;
        }
        w += __shfl_sync(0xffffffffu, cs, 31);
        u += __shfl_sync(0xffffffffu, us, 31);
      }
      if (pass == 0) {
        for (int o = 16; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        rt = most > 128 && w >= kLongChunks * (int)gridDim.x ? 256 : 128;
      }
    }
    if (lane == 0) {
      total[0] = w;
      total[1] = rt;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  const int W = total[0], rt = total[1];
  const uint32_t tmem = *tmem_slot;
  // With fewer chunks than CTAs the first W have one each: no CTA between a unit's first and
  // last is without a part of it.
  const int C = min((int)gridDim.x, W);
  const bool idle = (int)blockIdx.x >= C;
  const int c0 = idle ? 0 : cta_start(blockIdx.x, W, C);
  const int c1 = idle ? 0 : cta_start(blockIdx.x + 1, W, C);
  if (blockIdx.x == 0) {   // what own_kernel needs to find the partials
    if (tid == 0) {
      tp.plan[0] = W;
      tp.plan[1] = rt;
    }
    for (int g = tid; g < p.G; g += kThreads) {
      int4 v = make_int4(gr.start[g], gr.unit[g], (gr.s[g] + kChunk - 1) / kChunk, gr.rows[g]);
      reinterpret_cast<int4*>(tp.plan + 8)[g] = v;
    }
  }
  const bool wide = rt == 256;   // both streams serve every chunk
  int g = 0;
  if (c0 < c1) {                 // the first group of the range
    int a = 0, z = p.G;
    while (z - a > 1) {
      const int mid = (a + z) >> 1;
      if (gr.start[mid] <= c0) a = mid; else z = mid;
    }
    g = a;
  }
  Segment sg;
  int c = c0;

  if (warp == 8) {
    // ---- TMA producer: lane i brings page i of the chunk ----
    const int box = min(p.P, kChunk), ppc = kChunk / box;   // box rows, boxes per chunk
    int cnt = 0;
    while (next_segment(tp, gr, rt, c, c1, g, sg)) {
      const int32_t* row = p.block_table + (long long)sg.leader * p.max_pages;
      auto page_at = [&](int ch) -> int {
        const int tok = (sg.ch0 + ch) * kChunk + lane * box;
        return ch < sg.n && lane < ppc && tok < sg.s ? row[tok / p.P] : 0;
      };
      int next = page_at(0);
      for (int j = 0; j < sg.n; ++j, ++cnt) {
        const int st = cnt % NS;
        const uint32_t par = ((cnt / NS) & 1) ^ 1;
        const int t0 = (sg.ch0 + j) * kChunk;
        const int boxes = min(ppc, (sg.s - t0 + box - 1) / box);
        int page = next;
        next = page_at(j + 1);
        if (page < 0 || page >= p.num_pages) {
          atomicOr(p.status, kStatusBadPage);
          page = 0;
        }
        const int y = (int)(((long long)page * p.Hkv + sg.hk) * p.P + (t0 + lane * box) % p.P);
        const uint32_t bytes = (uint32_t)(boxes * box * D * 2);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t full = (kv ? vfull : kfull) + 8 * st, empty = (kv ? vempty : kempty) + 8 * st;
          mbar_wait_bounded(empty, par, abort_flag, p.status);
          const bool go = !*abort_flag;
          if (lane == 0 && go) mbar_arrive_expect_tx(full, bytes);
          __syncwarp();
          if (go && lane < boxes) {
            const uint32_t dst = sb + (kv ? S::kV : S::kK) + st * S::kOperand + lane * box * 128;
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
              tma_load_2d(dst + h * S::kTile, kv ? &map_v : &map_k, h * 64, y, full);
          }
          __syncwarp();
        }
      }
    }
    if (*abort_flag) {   // let the copies in flight land before the block goes
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {
      }
    }
  } else if (warp == 9) {
    // ---- tcgen05 issuer ----
    if (lane == 0) {
      int cnt = 0, nseg = 0, items_s[2] = {0, 0};
      while (next_segment(tp, gr, rt, c, c1, g, sg)) {
        const int items = wide ? 2 * sg.n : sg.n;
        mbar_wait_bounded(qready, nseg & 1, abort_flag, p.status);
        fence_after();
        auto issue_s = [&](int i) {   // S of item i: stream i & 1
          const int s = i & 1, ch = wide ? i >> 1 : i, k = cnt + ch, st = k % NS;
          if (!wide || s == 0) mbar_wait_bounded(kfull + 8 * st, (k / NS) & 1, abort_flag, p.status);
          fence_after();
          const uint32_t a = sb + S::kQ + (wide ? s : 0) * S::kOperand;
          const uint32_t b = sb + S::kK + st * S::kOperand;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk / 4) * S::kTile + (kk % 4) * 32;
            mma_ss(tmem + s * 128, desc_kmajor(a + off), desc_kmajor(b + off), ID_S, kk > 0);
          }
          commit(sfull + 8 * s);
          if (!wide || s == 1) commit(kempty + 8 * st);
        };
        issue_s(0);
        if (items > 1) issue_s(1);
        for (int i = 0; i < items; ++i) {
          const int s = i & 1, ch = wide ? i >> 1 : i, k = cnt + ch, st = k % NS;
          mbar_wait_bounded(pready + 8 * s, items_s[s] & 1, abort_flag, p.status);
          ++items_s[s];
          if (!wide || s == 0) mbar_wait_bounded(vfull + 8 * st, (k / NS) & 1, abort_flag, p.status);
          fence_after();
          const uint32_t b = sb + S::kV + st * S::kOperand;
#pragma unroll
          for (int kk = 0; kk < kChunk / 16; ++kk)
            mma_ts(tmem + 256 + s * D, tmem + s * 128 + kk * 8, desc_mnmajor(b + kk * 2048), ID_O,
                   i >= 2 || kk > 0);
          if (!wide || s == 1) commit(vempty + 8 * st);
          if (i + 2 >= items) commit(ofull + 8 * s);
          if (i + 2 < items) issue_s(i + 2);
        }
        cnt += sg.n;
        ++nseg;
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: thread = query row ----
    const int s = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + s * 128, to = tmem + lanes + 256 + s * D;
    const float kNegInf = __int_as_float(0xff800000);
    const float sc = fabsf(p.scale_log2);
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;   // the sign goes into q
    int cnt = 0, n_items = 0, n_o = 0;
    while (next_segment(tp, gr, rt, c, c1, g, sg)) {
      const int row = (wide ? s * 128 : 0) + r;        // row of the tile
      const bool warp_on = (wide ? s * 128 : 0) + (warp & 3) * 32 < sg.rows;
      // Q tile(s) into the swizzled operand layout; stream s loads its tile, or half of
      // the only one.  A 16-byte vector c of row x sits at x * 128 + ((c ^ x) & 7) * 16.
      bar_softmax();                                   // the exchange area is free again
      {
        constexpr int VPR = D / 8;                     // vectors of a row
        const uint32_t q0 = sb + S::kQ + (wide ? s * S::kOperand : 0);
        const int nv = 128 * VPR;
        const int first = wide ? r : tid, step = wide ? 128 : 256;
        for (int v = first; v < nv; v += step) {
          const int x = v / VPR, cv = v - x * VPR;
          const int qr = (wide ? s * 128 : 0) + x;
          uint4 val = make_uint4(0u, 0u, 0u, 0u);
          if (qr < sg.rows) {
            const int gr_row = sg.tile * rt + qr;
            const int b = sg.lo + gr_row / p.R, h = sg.hk * p.R + gr_row % p.R;
            val = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) +
                                                       ((long long)b * p.Hq + h) * D) + cv);
            val.x ^= flip; val.y ^= flip; val.z ^= flip; val.w ^= flip;
          }
          const uint32_t dst = q0 + (cv >> 3) * S::kTile + x * 128 + (((cv ^ x) & 7) << 4);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(val.x),
                       "r"(val.y), "r"(val.z), "r"(val.w)
                       : "memory");
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(qready);
      const int mine = wide ? sg.n : (sg.n - s + 1) / 2;   // items of this stream
      float m = kNegInf, l0 = 0.f, l1 = 0.f;
      for (int i = 0; i < mine; ++i, ++n_items) {
        const int ch = wide ? i : 2 * i + s;
        const int t0 = (sg.ch0 + ch) * kChunk;
        const int valid = min(kChunk, sg.s - t0);
        mbar_wait_bounded(sfull + 8 * s, n_items & 1, abort_flag, p.status);
        fence_after();
        if (valid < kChunk && (!wide || s == 0)) {
          // Rows of V behind the prefix hold anything; a weight 0 would not silence a NaN.
          // S of this item follows the products of the stream's item before, so the stage's
          // earlier chunk is done and the wait below cannot take its phase for this one.
          const int k = cnt + ch, st = k % NS;
          mbar_wait_bounded(vfull + 8 * st, (k / NS) & 1, abort_flag, p.status);
          const uint32_t v0 = sb + S::kV + st * S::kOperand;
          for (int q = r; q < (kChunk - valid) * 8 * S::kHalves; q += 128) {
            const int h = q / ((kChunk - valid) * 8), w = q - h * (kChunk - valid) * 8;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             v0 + h * S::kTile + valid * 128 + w * 16),
                         "r"(0u)
                         : "memory");
          }
          fence_proxy_async_smem();
        }
        if (warp_on) {
          float mx = kNegInf;
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            uint32_t v[32];
            ld32(ts + 32 * j, v);
            wait_ld();
            if (valid == kChunk) {
#pragma unroll
              for (int q = 0; q < 32; ++q) mx = fmaxf(mx, __uint_as_float(v[q]));
            } else {
#pragma unroll
              for (int q = 0; q < 32; ++q)
                if (32 * j + q < valid) mx = fmaxf(mx, __uint_as_float(v[q]));
            }
          }
          // Raise the reference maximum when the weights would pass 2^8.
          const bool first = i == 0;
          const bool raise = first || (mx - m) * sc > 8.f;
          if (__any_sync(0xffffffffu, raise)) {
            float f = 1.f;
            if (raise) {
              f = first ? 0.f : ex2((m - mx) * sc);
              if (m == kNegInf) f = 0.f;
              m = mx;
              l0 *= f;
              l1 *= f;
            }
            if (!first) {
#pragma unroll 1
              for (int j = 0; j < D / 32; ++j) {
                uint32_t v[32];
                ld32(to + 32 * j, v);
                wait_ld();
#pragma unroll
                for (int q = 0; q < 32; ++q) v[q] = __float_as_uint(__uint_as_float(v[q]) * f);
                st32(to + 32 * j, v);
              }
            }
          }
          const float ms = m == kNegInf ? 0.f : m * sc;
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            uint32_t v[32], w[16];
            ld32(ts + 32 * j, v);
            wait_ld();
#pragma unroll
            for (int q = 0; q < 32; q += 2) {
              float a = ex2(fmaf(__uint_as_float(v[q]), sc, -ms));
              float b = ex2(fmaf(__uint_as_float(v[q + 1]), sc, -ms));
              if (valid < kChunk) {
                if (32 * j + q >= valid) a = 0.f;
                if (32 * j + q + 1 >= valid) b = 0.f;
              }
              l0 += a;
              l1 += b;
              w[q / 2] = Mma<T>::pack(a, b);
            }
            // P's columns 16 j .. 16 j + 15 lie over S's columns of blocks <= j, read above.
            st16(ts + 16 * j, w);
          }
          wait_st();
        }
        fence_before();
        mbar_arrive(pready + 8 * s);
      }
      // ---- segment end ----
      const int slot = sg.unit + (int)blockIdx.x;
      const int rs = wide ? tp.rs_b : tp.rs_a;
      float4* po = reinterpret_cast<float4*>(p.part_o) + (long long)slot * rs * (D / 4);
      float* pl = p.part_lse + (long long)slot * rs;
      if (mine > 0) {
        mbar_wait_bounded(ofull + 8 * s, n_o & 1, abort_flag, p.status);
        ++n_o;
        fence_after();
      }
      float l = l0 + l1;
      const float ms = m == kNegInf ? 0.f : m * sc;    // log2 units
      if (wide) {
        if (warp_on) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
          for (int j = 0; j < D / 32; ++j) {
            uint32_t v[32];
            ld32(to + 32 * j, v);
            wait_ld();
            if (row < sg.rows) {
#pragma unroll
              for (int q = 0; q < 32; q += 4)
                po[(long long)(8 * j + q / 4) * rs + row] = make_float4(
                    __uint_as_float(v[q]) * inv, __uint_as_float(v[q + 1]) * inv,
                    __uint_as_float(v[q + 2]) * inv, __uint_as_float(v[q + 3]) * inv);
            }
          }
          if (row < sg.rows) pl[row] = l == 0.f ? kNegInf : ms + log2f(l);
        }
      } else {
        // Each stream finishes half of the columns: it hands the other half of its O over.
        float* xo = reinterpret_cast<float*>(smem + S::kQ) + s * (D / 2) * 128;
        ml[s * 128 + r] = make_float2(ms, mine > 0 ? l : 0.f);
        if (warp_on && mine > 0) {
#pragma unroll 1
          for (int j = 0; j < D / 64; ++j) {
            uint32_t v[32];
            ld32(to + (1 - s) * (D / 2) + 32 * j, v);
            wait_ld();
#pragma unroll
            for (int q = 0; q < 32; ++q) xo[(32 * j + q) * 128 + r] = __uint_as_float(v[q]);
          }
        }
        bar_softmax();
        if (warp_on) {
          const float2 other = ml[(1 - s) * 128 + r];
          const float lo_ = other.y;
          const bool have_o = (sg.n - (1 - s) + 1) / 2 > 0;    // the other stream had items
          const float M = l == 0.f ? other.x : lo_ == 0.f ? ms : fmaxf(ms, other.x);
          const float wa = l == 0.f ? 0.f : ex2(ms - M), wb = lo_ == 0.f ? 0.f : ex2(other.x - M);
          const float L = l * wa + lo_ * wb;
          const float inv = L == 0.f ? 0.f : 1.f / L;
          const float ia = wa * inv, ib = wb * inv;
          const float* yo = reinterpret_cast<const float*>(smem + S::kQ) + (1 - s) * (D / 2) * 128;
#pragma unroll 1
          for (int j = 0; j < D / 64; ++j) {
            uint32_t v[32];
            if (mine > 0) {
              ld32(to + s * (D / 2) + 32 * j, v);
              wait_ld();
            }
            if (row < sg.rows) {
#pragma unroll
              for (int q = 0; q < 32; q += 4) {
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  o[e] = mine > 0 ? __uint_as_float(v[q + e]) * ia : 0.f;
                  if (have_o) o[e] = fmaf(yo[(32 * j + q + e) * 128 + r], ib, o[e]);
                }
                po[(long long)(s * (D / 8) + 8 * j + q / 4) * rs + row] =
                    make_float4(o[0], o[1], o[2], o[3]);
              }
            }
          }
          if (s == 0 && row < sg.rows) pl[row] = L == 0.f ? kNegInf : M + log2f(L);
        }
      }
      fence_before();   // O is read: the next segment's products may overwrite it
      cnt += sg.n;
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
// own_kernel: a sequence's own tokens and the join.
//
// Block = (token split, KV head and 8 * NH query heads, sequence), four warps, each with
// 16 tokens at a time and a softmax state of its own.  Nothing is staged in shared memory:
//   S[heads x tokens] = Q K^T by mma.m16n8k16 with the head-size index permuted, so that a
//   thread's share of a key row is whole 16-byte vectors (Q is loaded the same way);
//   O^T[d x heads] += V^T P^T: a thread's vectors of two tokens, interleaved by byte
//   permutes, are V^T's fragment, again with d permuted (the output index follows), and
//   P^T's fragment is S's accumulator itself.
// The splits of a sequence are a cluster; warps, splits and the prefix's partials are
// joined per output element by the blocks of the cluster together.
template <int D, int NH>
struct OwnSmem {
  static constexpr int kHeads = 8 * NH;
  static constexpr int kWarps = 4;
  static constexpr int kO = 0;                                    // [4][heads][D] fp32
  static constexpr int kMl = kO + kWarps * kHeads * D * 4;        // [4][heads] (max, sum)
  static constexpr int kInfo = kMl + kWarps * kHeads * 8;         // per head: M, 1 / L
  static constexpr int kBytes = kInfo + kHeads * 8;
};

__device__ __forceinline__ uint32_t own_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void own_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ uint32_t own_map(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 own_ld2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 own_ld4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

template <int D, int NH, typename T>
__global__ void __launch_bounds__(128) own_kernel(const __grid_constant__ TcParams tp) {
  using SM = OwnSmem<D, NH>;
  constexpr int HEADS = SM::kHeads;
  constexpr int NK = D / 32;     // 16-byte vectors of a key row per thread
  constexpr int NV = D / 64;     // of a value row per thread
  const Params& p = tp.p;
  __shared__ __align__(16) uint8_t sm[SM::kBytes];
  __shared__ int scratch[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, t4 = lane & 3;
  const int ns = gridDim.x, split = blockIdx.x;
  const int hgs = (p.R + HEADS - 1) / HEADS;
  const int hk = blockIdx.y / hgs, hg = blockIdx.y - hk * hgs;
  const int b = blockIdx.z;
  const int h0 = hk * p.R + hg * HEADS;                  // first query head
  const int nh = min(HEADS, p.R - hg * HEADS);
  const float kNegInf = __int_as_float(0xff800000);
  pdl_launch_dependents();
  // Everything up to the join reads only what was final before prefix_kernel let this
  // kernel start (it does so behind its own wait for its predecessors).

  const int g = group_of(p, b, scratch);
  int s = 0, lo = 0;
  if (g >= 0) {
    int hi, leader;
    group_range(p, g, lo, hi);
    group_prefix(p, g, lo, hi, scratch, s, leader);
  }
  const int len = seq_len(p, b, split == 0 && tid == 0);
  bool shared = s > 0 && len > 0;
  const int t_begin = min(s, len);

  // Q: rows gq and gq + 8 of the m16 tile are heads of this block.
  uint32_t qa[2 * NK][4];
  {
    const T* q = reinterpret_cast<const T*>(p.q) + ((long long)b * p.Hq + h0) * D;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
      if (gq < nh) x = __ldg(reinterpret_cast<const uint4*>(q + gq * D) + i * 4 + t4);
      if (NH == 2 && gq + 8 < nh)
        y = __ldg(reinterpret_cast<const uint4*>(q + (gq + 8) * D) + i * 4 + t4);
      qa[2 * i][0] = x.x; qa[2 * i][2] = x.y; qa[2 * i + 1][0] = x.z; qa[2 * i + 1][2] = x.w;
      qa[2 * i][1] = y.x; qa[2 * i][3] = y.y; qa[2 * i + 1][1] = y.z; qa[2 * i + 1][3] = y.w;
    }
  }
  float m[NH], l[NH], o[NH][D / 16][4];
#pragma unroll
  for (int a = 0; a < NH; ++a) {
    m[a] = kNegInf;
    l[a] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[a][j][e] = 0.f;
  }
  const T* kp = reinterpret_cast<const T*>(p.k_pages);
  const T* vp = reinterpret_cast<const T*>(p.v_pages);
  const int32_t* row = p.block_table + (long long)b * p.max_pages;
  const int stride = 16 * 4 * ns;
  for (int t0 = t_begin + 16 * (split * 4 + warp); t0 < len; t0 += stride) {
    // Rows of this thread: keys t0 + gq, t0 + gq + 8; values t0 + {2 t4, 2 t4 + 1, + 8, + 9}.
    auto base_of = [&](int tok) -> long long {
      int page = row[tok / p.P];
      if (page < 0 || page >= p.num_pages) {
        atomicOr(p.status, kStatusBadPage);
        page = 0;
      }
      return (((long long)page * p.Hkv + hk) * p.P + tok % p.P) * D;
    };
    uint4 kx[2][NK], vx[4][NV];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const int tok = t0 + gq + 8 * a;
#pragma unroll
      for (int i = 0; i < NK; ++i) kx[a][i] = make_uint4(0u, 0u, 0u, 0u);
      if (tok < len) {
        const uint4* src = reinterpret_cast<const uint4*>(kp + base_of(tok)) + t4;
#pragma unroll
        for (int i = 0; i < NK; ++i) kx[a][i] = __ldg(src + i * 4);
      }
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int tok = t0 + 2 * t4 + (a & 1) + 8 * (a >> 1);
#pragma unroll
      for (int i = 0; i < NV; ++i) vx[a][i] = make_uint4(0u, 0u, 0u, 0u);
      if (tok < len) {
        const uint4* src = reinterpret_cast<const uint4*>(vp + base_of(tok)) + gq;
#pragma unroll
        for (int i = 0; i < NV; ++i) vx[a][i] = __ldg(src + i * 8);
      }
    }
    float sc[2][4];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[a][e] = 0.f;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        Mma<T>::run(sc[a], qa[2 * i], kx[a][i].x, kx[a][i].y);
        Mma<T>::run(sc[a], qa[2 * i + 1], kx[a][i].z, kx[a][i].w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)   // tokens t0 + 8 a + 2 t4 + (e & 1)
        sc[a][e] = t0 + 8 * a + 2 * t4 + (e & 1) < len ? sc[a][e] * p.scale_log2 : kNegInf;
    }
#pragma unroll
    for (int a = 0; a < NH; ++a) {
      // heads gq + 8 a
      float tm = fmaxf(fmaxf(sc[0][2 * a], sc[0][2 * a + 1]), fmaxf(sc[1][2 * a], sc[1][2 * a + 1]));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 1));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 2));
      const float mn = fmaxf(m[a], tm);
      const float mu = mn == kNegInf ? 0.f : mn;
      const float f = ex2(m[a] - mu);
      m[a] = mn;
      const float p0 = ex2(sc[0][2 * a] - mu), p1 = ex2(sc[0][2 * a + 1] - mu);
      const float p2 = ex2(sc[1][2 * a] - mu), p3 = ex2(sc[1][2 * a + 1] - mu);
      l[a] = l[a] * f + ((p0 + p1) + (p2 + p3));
      const uint32_t b0 = Mma<T>::pack(p0, p1), b1 = Mma<T>::pack(p2, p3);
      if (__any_sync(0xffffffffu, f != 1.f)) {
        const float f0 = __shfl_sync(0xffffffffu, f, 8 * t4), f1 = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[a][j][0] *= f0; o[a][j][1] *= f1; o[a][j][2] *= f0; o[a][j][3] *= f1;
        }
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const int i = j / 4, w = j % 4;
        auto word = [&](const uint4& v) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; };
        uint32_t af[4];
        af[0] = __byte_perm(word(vx[0][i]), word(vx[1][i]), 0x5410);
        af[1] = __byte_perm(word(vx[0][i]), word(vx[1][i]), 0x7632);
        af[2] = __byte_perm(word(vx[2][i]), word(vx[3][i]), 0x5410);
        af[3] = __byte_perm(word(vx[2][i]), word(vx[3][i]), 0x7632);
        Mma<T>::run(o[a][j], af, b0, b1);
      }
    }
  }
  // ---- this warp's state into shared memory ----
  float* so = reinterpret_cast<float*>(sm + SM::kO) + warp * HEADS * D;
  float2* sml = reinterpret_cast<float2*>(sm + SM::kMl) + warp * HEADS;
#pragma unroll
  for (int a = 0; a < NH; ++a) {
    float ls = l[a];
    ls += __shfl_xor_sync(0xffffffffu, ls, 1);
    ls += __shfl_xor_sync(0xffffffffu, ls, 2);
    if (t4 == 0) sml[8 * a + gq] = make_float2(m[a], ls);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      // rows gq, gq + 8 of the m-tile are d, d + 1; columns are heads 2 t4, 2 t4 + 1
      const int d = (j / 4) * 64 + gq * 8 + 2 * (j % 4);
      *reinterpret_cast<float2*>(so + (8 * a + 2 * t4) * D + d) = make_float2(o[a][j][0], o[a][j][2]);
      *reinterpret_cast<float2*>(so + (8 * a + 2 * t4 + 1) * D + d) = make_float2(o[a][j][1], o[a][j][3]);
    }
  }
  // ---- join: warps and splits of the cluster, then the prefix's partials ----
  if (ns > 1) own_cluster_sync(); else __syncthreads();
  pdl_wait();   // prefix_kernel's partials and plan
  const uint32_t a_o = smem_u32(sm + SM::kO), a_ml = smem_u32(sm + SM::kMl);
  int first = 0, nseg = 0, W = 0, rt = 128, rs = 1, unit0 = 0, start = 0, nch = 0, tiles = 1;
  if (shared) {
    W = tp.plan[0];
    rt = tp.plan[1];
    const int4 v = reinterpret_cast<const int4*>(tp.plan + 8)[g];
    start = v.x; unit0 = v.y; nch = v.z;
    shared = nch > 0;   // bad groups (reported): prefix_kernel has left nothing
    tiles = (v.w + rt - 1) / rt;
    rs = rt == 256 ? tp.rs_b : tp.rs_a;
  }
  // A thread makes 4 elements of a head at a time, the blocks of a cluster share the heads.
  const int items = nh * (D / 4);
  for (int it = split * 128 + tid; it < items; it += ns * 128) {
    const int h = it / (D / 4), d4 = it - h * (D / 4);
    float M = kNegInf;
    for (int e = 0; e < 4 * ns; ++e) {
      const float2 v = own_ld2(own_map(a_ml + ((e & 3) * HEADS + h) * 8, e >> 2));
      if (v.y != 0.f) M = fmaxf(M, v.x);
    }
    long long slot0 = 0;
    if (shared) {
      const int rr = (b - lo) * p.R + hg * HEADS + h;      // row of the group
      const int tile = rr / rt, u = hk * tiles + tile;
      const int ustart = start + u * nch;
      const int C = min(tp.ctas, W);
      first = cta_owner(ustart, W, C);
      nseg = cta_owner(ustart + nch - 1, W, C) - first + 1;
      slot0 = (long long)(unit0 + u + first);
      const float* pl = p.part_lse + slot0 * rs + (rr - tile * rt);
#pragma unroll 4
      for (int e = 0; e < nseg; ++e) M = fmaxf(M, pl[(long long)e * rs]);
    }
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const float mu = M == kNegInf ? 0.f : M;
    for (int e = 0; e < 4 * ns; ++e) {
      const float2 v = own_ld2(own_map(a_ml + ((e & 3) * HEADS + h) * 8, e >> 2));
      if (v.y == 0.f) continue;
      const float w = ex2(v.x - mu);
      const float4 x = own_ld4(own_map(a_o + (((e & 3) * HEADS + h) * D + d4 * 4) * 4, e >> 2));
      L = fmaf(v.y, w, L);
      acc.x = fmaf(x.x, w, acc.x); acc.y = fmaf(x.y, w, acc.y);
      acc.z = fmaf(x.z, w, acc.z); acc.w = fmaf(x.w, w, acc.w);
    }
    if (shared) {
      const int rr = (b - lo) * p.R + hg * HEADS + h;
      const int tr = rr - rr / rt * rt;
      const float* pl = p.part_lse + slot0 * rs + tr;
      const float4* po = reinterpret_cast<const float4*>(p.part_o) +
                         (slot0 * (D / 4) + d4) * rs + tr;
#pragma unroll 4
      for (int e = 0; e < nseg; ++e) {
        const float w = ex2(pl[(long long)e * rs] - mu);   // an empty part: 2^-inf = 0
        const float4 x = po[(long long)e * rs * (D / 4)];
        L += w;
        acc.x = fmaf(x.x, w, acc.x); acc.y = fmaf(x.y, w, acc.y);
        acc.z = fmaf(x.z, w, acc.z); acc.w = fmaf(x.w, w, acc.w);
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;     // an empty sequence gives zeros
    uint2 r;
    r.x = Mma<T>::pack(acc.x * inv, acc.y * inv);
    r.y = Mma<T>::pack(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + ((long long)b * p.Hq + h0 + h) * D +
                              d4 * 4) = r;
  }
  if (ns > 1) own_cluster_sync();   // the peers have read this block's shared memory
}

}  // namespace tc
}  // namespace prefix
}  // namespace llmc
