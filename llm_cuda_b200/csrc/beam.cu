// Beam search over the paged cache: the selection of a step and the reordering after it.
//
// beam_select: for every prompt, the n best of
//     score[k, v] = beam_score[k] + (x[k, v] - lse(x[k, :]))
// over its K beams and the vocabulary, in descending order, ties to the lowest k * V + v.
// One launch and no global workspace: a thread-block cluster owns a prompt and cuts its
// K rows into tasks (row, split).  A task is one pass over its logits: every thread keeps
// a running maximum and sum of exponentials, every warp the n best logits it has seen (a
// threshold and a short list in shared memory, so an element usually costs one compare).
// The order inside a row is that of its logits, which needs no log-sum-exp, so one pass is
// enough.  The CTA merges its warps' lists by rank, the cluster's first CTA collects all
// lists and sums through distributed shared memory and ranks the candidates by their
// scores.  Bound: the logits are read once from HBM.
//
// Sums of exponentials are held in fp32 per thread and joined in fp64; scores are ranked
// in fp64 (candidates of different beams are often closer than fp32 tells apart) and
// rounded once to fp32.
//
// beam_reorder: beam i of a prompt continues from beam parent[i].  See below.
#include <climits>
#include <string>

#include "common.cuh"

namespace llmc {
namespace beam {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBeams = 32;
constexpr int kU = 4;           // 16-byte vectors a lane has in flight

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ uint32_t dsmem_addr(uint32_t local_addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_addr), "r"(rank));
  return remote;
}
__device__ __forceinline__ unsigned long long ld_dsmem_u64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// Order-preserving bits of a float, then the complemented index: larger is better, equal
// values rank by the lowest index.  Never zero for a number (0 means "no entry").
__device__ __forceinline__ unsigned long long make_key(float f, uint32_t idx) {
  uint32_t u = __float_as_uint(f);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}
__device__ __forceinline__ uint32_t key_index(unsigned long long k) {
  return 0xFFFFFFFFu - (uint32_t)k;
}

struct SelectParams {
  const void* logits;
  long long row_stride;      // elements between rows
  const float* beam_scores;  // [G, K]
  const uint8_t* finished;   // [G, K] or NULL
  float* out_scores;         // [G, n]
  int32_t* out_beams;
  int64_t* out_tokens;
  int K, V, n, eos, splits;  // splits: tasks of one row
};

// A warp's list of the n best logits seen so far: `count` keys in any order in shared
// memory.  Once it holds n, `tau` is the n-th best of them; elements of later tiles have
// larger indices, so only strictly larger values pass (`full`).
constexpr int kCap = 128;   // n + 32 <= kCap

struct WarpTop {
  unsigned long long* buf;
  int n, count;
  float tau;
  bool full;
};

// Sort the buffer by rank (keys are distinct), keep the first n.
__device__ __forceinline__ void top_compact(WarpTop& t, int lane) {
  constexpr int E = kCap / 32;
  __syncwarp();
  unsigned long long mine[E];
  int rank[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = lane + 32 * e;
    mine[e] = i < t.count ? t.buf[i] : 0ull;
    rank[e] = 0;
  }
  for (int j = 0; j < t.count; ++j) {
    const unsigned long long o = t.buf[j];
#pragma unroll
    for (int e = 0; e < E; ++e) rank[e] += o > mine[e] ? 1 : 0;
  }
  __syncwarp();
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + 32 * e < t.count && rank[e] < t.n) t.buf[rank[e]] = mine[e];
  __syncwarp();
  if (t.count >= t.n) {
    t.count = t.n;
    t.tau = key_value(t.buf[t.n - 1]);
    t.full = true;
  }
}

// The n-th largest of the lanes' values (n <= 32): a bitonic sort across the warp.
__device__ __forceinline__ float nth_lane_max(float v, int n, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j; j >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, j);
      const bool up = ((lane & k) == 0) == ((lane & j) == 0);   // descending
      v = up ? fmaxf(v, o) : fminf(v, o);
    }
  }
  return __shfl_sync(0xffffffffu, v, n - 1);
}

// 2^x by the hardware (2 ulp); exp2f adds a range check for results below 2^-126, which
// a sum whose largest term is 1 does not notice.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) beam_select_kernel(const SelectParams p) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t sm_raw[];
  const int n = p.n, K = p.K, V = p.V, S = p.splits;
  const uint32_t rank = cluster_ctarank(), C = cluster_nctarank();
  const int g = blockIdx.x / C;
  const int tasks = K * S;
  const int per_cta = (tasks + (int)C - 1) / (int)C;
  // shared: warp buffers [kWarps][kCap], this CTA's lists [per_cta][n], sums [per_cta],
  // then (first CTA) all lists [tasks][n], row constants.
  unsigned long long* wbuf = reinterpret_cast<unsigned long long*>(sm_raw);
  unsigned long long* lists = wbuf + kWarps * kCap;
  unsigned long long* sums = lists + (size_t)per_cta * n;       // (max, sum) as two floats
  unsigned long long* all = sums + per_cta;
  double* row_lse = reinterpret_cast<double*>(all + (size_t)tasks * n);
  double* row_b = row_lse + K;
  int* row_kind = reinterpret_cast<int*>(row_b + K);            // 0 live, 1 dead, 2 finished
  __shared__ float red_m[kWarps], red_s[kWarps];
  __shared__ int wcount[kWarps];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();

  constexpr float kLog2e = 1.4426950408889634f;
  const float kNegInf = __int_as_float(0xff800000);

  for (int t = (int)rank, slot = 0; t < tasks; t += (int)C, ++slot) {
    const int row = t / S, split = t - row * S;
    const bool fin = p.finished && p.finished[(long long)g * K + row];
    unsigned long long* out = lists + (size_t)slot * n;
    if (fin) {   // offers eos alone: its logits are not read
      for (int i = threadIdx.x; i < n; i += kThreads) out[i] = 0ull;
      if (threadIdx.x == 0) sums[slot] = 0ull;
      continue;
    }
    const T* x = reinterpret_cast<const T*>(p.logits) + ((long long)g * K + row) * p.row_stride;
    // Vectors are 16-byte aligned: vector v holds elements [v * VEC - h, v * VEC - h + VEC).
    const int h = (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % VEC);
    const int nvec = (V + h + VEC - 1) / VEC;
    const int v0 = (int)((long long)nvec * split / S), v1 = (int)((long long)nvec * (split + 1) / S);
    // A warp's vectors are contiguous, so its later elements have larger indices.
    const int w0 = v0 + (int)((long long)(v1 - v0) * warp / kWarps);
    const int w1 = v0 + (int)((long long)(v1 - v0) * (warp + 1) / kWarps);
    WarpTop top;
    top.buf = wbuf + warp * kCap;
    top.n = n;
    top.count = 0;
    top.tau = kNegInf;
    top.full = false;
    float m = kNegInf, s = 0.f;
    bool nan = false;
    for (int base = w0; base < w1; base += 32 * kU) {
      uint4 raw[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int v = base + u * 32 + lane;
        const long long e0 = (long long)v * VEC - h;
        T* r = reinterpret_cast<T*>(&raw[u]);
        if (v < w1 && e0 >= 0 && e0 + VEC <= V) {
          raw[u] = __ldg(reinterpret_cast<const uint4*>(x + e0));
        } else {   // the ends of a row, or past this warp's part: -inf outside
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            r[e] = (v < w1 && e0 + e >= 0 && e0 + e < V) ? x[e0 + e] : from_f32<T>(kNegInf);
        }
      }
      float tile_m = kNegInf;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const T* r = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) tile_m = fmaxf(tile_m, to_f32(r[e]));
      }
      // running maximum and sum of this thread
      if (tile_m > m) {
        s *= ex2((m - tile_m) * kLog2e);   // m = -inf: s is 0
        m = tile_m;
      }
      const float mm = m == kNegInf ? 0.f : m;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const T* r = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += ex2((to_f32(r[e]) - mm) * kLog2e);
      }
      nan |= s != s;
      // The n best: nothing to do unless some lane's largest value passes.
      if (top.full && !__any_sync(0xffffffffu, tile_m > top.tau)) continue;
      // Before the list is full, the n-th largest lane maximum bounds the tile's n-th best.
      const float lo = top.full ? top.tau : (n <= 32 ? nth_lane_max(tile_m, n, lane) : kNegInf);
      uint32_t mask = 0;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int v = base + u * 32 + lane;
        const T* r = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const long long i = (long long)v * VEC - h + e;
          const float f = to_f32(r[e]);
          const bool pass = (top.full ? f > lo : f >= lo) && v < w1 && i >= 0 && i < V;
          mask |= pass ? 1u << (u * VEC + e) : 0u;
        }
      }
      while (true) {
        bool pass = mask != 0;
        unsigned vote = __ballot_sync(0xffffffffu, pass);
        if (!vote) break;
        const int bit = pass ? __ffs(mask) - 1 : 0;
        mask &= mask - 1;
        float f = 0.f;
#pragma unroll
        for (int q = 0; q < kU * VEC; ++q)
          if (q == bit) f = to_f32(reinterpret_cast<const T*>(&raw[q / VEC])[q % VEC]);
        if (top.count + __popc(vote) > kCap) {
          // Elements of this tile are in no order: equal values still compete by index.
          top_compact(top, lane);
          pass = pass && (!top.full || f >= top.tau);
          vote = __ballot_sync(0xffffffffu, pass);
        }
        const int v = base + (bit / VEC) * 32 + lane;
        if (pass)
          top.buf[top.count + __popc(vote & ((1u << lane) - 1u))] =
              make_key(f, (uint32_t)((long long)v * VEC - h + bit % VEC));
        top.count += __popc(vote);
      }
      if (!top.full && top.count >= n) top_compact(top, lane);
    }
    top_compact(top, lane);
    // join the warps: maximum and sum, then the lists
    if (nan) s = __int_as_float(0x7fc00000);   // a NaN, or an infinity, among the logits
    float wm = m;
    for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
    float ws = m == kNegInf ? s : s * ex2((m - wm) * kLog2e);
    for (int o = 16; o; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
    if (lane == 0) {
      red_m[warp] = wm;
      red_s[warp] = ws;
      wcount[warp] = top.count;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      float M = kNegInf;
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, red_m[w]);
      float sum = 0.f;
      for (int w = 0; w < kWarps; ++w)
        sum += red_m[w] == kNegInf ? red_s[w] : red_s[w] * ex2((red_m[w] - M) * kLog2e);
      sums[slot] = ((unsigned long long)__float_as_uint(M) << 32) | __float_as_uint(sum);
    }
    for (int i = threadIdx.x; i < n; i += kThreads) out[i] = 0ull;
    __syncthreads();
    for (int i = threadIdx.x; i < kWarps * n; i += kThreads) {
      const int w = i / n, j = i - w * n;
      if (j >= wcount[w]) continue;
      const unsigned long long key = wbuf[w * kCap + j];
      int r = j;
      for (int q = 0; q < kWarps && r < n; ++q) {
        if (q == w) continue;
        // entries of the sorted list q that are better
        int lo = 0, hi = wcount[q];
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (wbuf[q * kCap + mid] > key) lo = mid + 1; else hi = mid;
        }
        r += lo;
      }
      if (r < n) out[r] = key;
    }
    __syncthreads();
  }
  cluster_sync_all();   // every list is written
  if (rank == 0) {
    // All lists and sums, from the CTA that made them.
    for (int i = threadIdx.x; i < tasks * n; i += kThreads) {
      const int t = i / n, j = i - t * n;
      all[i] = ld_dsmem_u64(dsmem_addr(smem_u32(lists + (size_t)(t / (int)C) * n + j),
                                       (uint32_t)(t % (int)C)));
    }
    for (int k = threadIdx.x; k < K; k += kThreads) {
      const long long gk = (long long)g * K + k;
      const float b = p.beam_scores[gk];
      double M = -INFINITY, sum = 0.0;
      for (int sp = 0; sp < S; ++sp) {
        const int t = k * S + sp;
        const unsigned long long u =
            ld_dsmem_u64(dsmem_addr(smem_u32(sums + t / (int)C), (uint32_t)(t % (int)C)));
        const double mt = (double)__uint_as_float((uint32_t)(u >> 32));
        const double st = (double)__uint_as_float((uint32_t)u);
        if (mt > M) {
          sum = (isinf(M) ? sum : sum * exp(M - mt)) + st;
          M = mt;
        } else {
          sum += isinf(mt) ? st : st * exp(mt - M);
        }
      }
      const double lse = M + log(sum);
      const bool fin = p.finished && p.finished[gk];
      row_b[k] = (double)b;
      row_lse[k] = lse;
      row_kind[k] = !isfinite(b) ? 1 : fin ? 2 : isfinite(lse) ? 0 : 1;
    }
  }
  cluster_sync_all();   // the peers' shared memory has been read
  if (rank != 0) return;
  __syncthreads();
  const int per_row = S * n;
  // Rows without usable scores offer their lowest tokens at -inf; finished rows eos first.
  for (int k = 0; k < K; ++k) {
    if (row_kind[k] == 0) continue;
    for (int i = threadIdx.x; i < per_row; i += kThreads) {
      unsigned long long key = 0ull;
      if (i < n) {
        if (row_kind[k] == 1) {
          if (i < V) key = make_key(kNegInf, (uint32_t)i);
        } else if (i == 0) {
          key = make_key(0.f, (uint32_t)p.eos);
        } else {
          const int tok = i - 1 < p.eos ? i - 1 : i;
          if (tok < V) key = make_key(kNegInf, (uint32_t)tok);
        }
      }
      all[(size_t)k * per_row + i] = key;
    }
  }
  __syncthreads();
  auto score_of = [&](int k, unsigned long long key) -> double {
    const float v = key_value(key);
    if (row_kind[k] == 1) return -INFINITY;
    if (row_kind[k] == 2) return v == 0.f ? row_b[k] : -INFINITY;
    return row_b[k] + ((double)v - row_lse[k]);
  };
  // Rank of every candidate: how many of the sorted lists' entries are better.
  for (int i = threadIdx.x; i < tasks * n; i += kThreads) {
    const unsigned long long key = all[i];
    if (key == 0ull) continue;
    const int t = i / n, j = i - t * n, k = t / S;
    const double sc = score_of(k, key);
    const long long flat = (long long)k * V + key_index(key);
    int r = j;
    for (int q = 0; q < tasks && r < n; ++q) {
      if (q == t) continue;
      const int kq = q / S;
      const unsigned long long* L = all + (size_t)q * n;
      int lo = 0, hi = n;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const unsigned long long o = L[mid];
        bool better = false;
        if (o != 0ull) {
          if (kq == k) {
            better = o > key;
          } else {
            const double so = score_of(kq, o);
            better = so > sc || (so == sc && (long long)kq * V + key_index(o) < flat);
          }
        }
        if (better) lo = mid + 1; else hi = mid;
      }
      r += lo;
    }
    if (r < n) {
      const long long o = (long long)g * n + r;
      p.out_scores[o] = (float)sc;
      p.out_beams[o] = k;
      p.out_tokens[o] = (int64_t)key_index(key);
    }
  }
}

// ---------------------------------------------------------------------------------
// Reordering.  Beam i of a prompt (K beams, all of one length L) continues from beam
// p = parent[i].  Every beam has its own page for each logical page behind the prompt
// (own_table); a beam writes only the page that holds position L, and only into its own.
// So full pages are never copied: row i of the block table takes the parent's entries for
// the logical pages below L / P and i's own ones from there on, and the L % P tokens of
// the page in progress are copied from p's own page to i's own page, in every layer.
//
// The copies of a prompt form a permutation with repeats, in place: a thread loads one
// 16-byte vector of all K pages, then stores them, so no copy sees another's result.  The
// table is moved the same way, a thread per column.  Bound: HBM (the moved tokens), and
// at small sizes the launch.
struct ReorderParams {
  uint8_t* pools;              // [layers][2][num_pages][Hkv][P][d]
  const int32_t* own_table;    // [G * K, max_pages]
  int32_t* block_table;
  const int32_t* seq_lens;     // [G * K]
  const int32_t* parents;      // [G, K]
  int32_t* status;
  long long pool_bytes;        // of one layer's K or V pool
  long long page_bytes;        // of one page (all heads)
  int head_bytes;              // P * d * element size
  int tok_bytes;               // d * element size
  int K, layers2, Hkv, P, max_pages, num_pages;
};

template <int KM, typename Vec>
__global__ void __launch_bounds__(256) beam_reorder_kernel(const ReorderParams p) {
  const int g = blockIdx.y, K = p.K;
  __shared__ int s_par[kMaxBeams], s_page[kMaxBeams], s_bad;
  pdl_launch_dependents();
  pdl_wait();
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  const long long b0 = (long long)g * K;
  const int len = p.seq_lens[b0];
  const int full = len >= 0 ? len / p.P : 0;
  const int fill = len >= 0 ? len - full * p.P : 0;
  if (threadIdx.x < K) {
    const int i = threadIdx.x;
    const int par = p.parents[b0 + i];
    int bad = 0;
    if (par < 0 || par >= K || p.seq_lens[b0 + i] != len) bad = kStatusBadParent;
    if (len < 0 || (long long)len > (long long)p.max_pages * p.P) bad |= kStatusSeqLenRange;
    int page = 0;
    if (!bad && fill) {
      page = p.own_table[(b0 + i) * p.max_pages + full];
      if (page < 0 || page >= p.num_pages) bad = kStatusBadPage;
    }
    if (bad) {
      atomicOr(&s_bad, bad);
      atomicOr(p.status, bad);
    }
    s_par[i] = par;
    s_page[i] = page;
  }
  __syncthreads();
  if (s_bad) return;   // a prompt with a bad entry is left as it is
  if ((int)blockIdx.x == p.layers2) {   // the table
    for (int c = blockIdx.z * blockDim.x + threadIdx.x; c < p.max_pages;
         c += gridDim.z * blockDim.x) {
      int32_t v[KM];
#pragma unroll
      for (int i = 0; i < KM; ++i)
        if (i < K)
          v[i] = c < full ? p.block_table[(b0 + s_par[i]) * p.max_pages + c]
                          : p.own_table[(b0 + i) * p.max_pages + c];
#pragma unroll
      for (int i = 0; i < KM; ++i)
        if (i < K) p.block_table[(b0 + i) * p.max_pages + c] = v[i];
    }
    return;
  }
  uint8_t* pool = p.pools + (long long)blockIdx.x * p.pool_bytes;
  const int vph = fill * (p.tok_bytes / (int)sizeof(Vec));   // vectors of one head
  const int total = p.Hkv * vph;
  for (int v = blockIdx.z * blockDim.x + threadIdx.x; v < total; v += gridDim.z * blockDim.x) {
    const int head = v / vph;
    const long long off = (long long)head * p.head_bytes + (long long)(v - head * vph) * sizeof(Vec);
    Vec r[KM];
#pragma unroll
    for (int i = 0; i < KM; ++i)
      if (i < K && s_par[i] != i)
        r[i] = *reinterpret_cast<const Vec*>(pool + s_page[s_par[i]] * p.page_bytes + off);
#pragma unroll
    for (int i = 0; i < KM; ++i)
      if (i < K && s_par[i] != i)
        *reinterpret_cast<Vec*>(pool + s_page[i] * p.page_bytes + off) = r[i];
  }
}

}  // namespace beam

template <typename T>
static cudaError_t launch_select_t(const beam::SelectParams& p0, int G, cudaStream_t stream) {
  beam::SelectParams p = p0;
  auto kern = beam::beam_select_kernel<T>;
  // CTAs per prompt: 16 while that leaves SMs idle, else 8 (the portable size).
  const int C = G <= 16 ? 16 : 8;
  p.splits = C / p.K > 1 ? C / p.K : 1;
  const int tasks = p.K * p.splits, per = (tasks + C - 1) / C;
  const size_t smem = sizeof(unsigned long long) *
                          ((size_t)beam::kWarps * beam::kCap + (size_t)per * p.n + per +
                           (size_t)tasks * p.n) +
                      (size_t)p.K * (2 * sizeof(double) + sizeof(int));
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess && C > 8)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(G * C));
  cfg.blockDim = dim3(beam::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kern, p);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_beam_select(const void* logits, long long row_stride, const float* beam_scores,
                               const uint8_t* finished, float* out_scores, int32_t* out_beams,
                               int64_t* out_tokens, int G, int K, int V, int n, int eos, int dtype,
                               cudaStream_t stream) {
  beam::SelectParams p;
  p.logits = logits; p.row_stride = row_stride; p.beam_scores = beam_scores;
  p.finished = finished; p.out_scores = out_scores; p.out_beams = out_beams;
  p.out_tokens = out_tokens;
  p.K = K; p.V = V; p.n = n; p.eos = eos; p.splits = 1;
  if (dtype == LLMC_F32) return launch_select_t<float>(p, G, stream);
  if (dtype == LLMC_F16) return launch_select_t<__half>(p, G, stream);
  return launch_select_t<__nv_bfloat16>(p, G, stream);
}

template <int KM>
static cudaError_t launch_reorder_k(const beam::ReorderParams& p, int G, bool vec16,
                                    cudaStream_t stream) {
  // Blocks along a pool's tokens: enough to fill the GPU when there are few prompts.
  const long long blocks = (long long)p.layers2 * G;
  const long long vecs = (long long)p.page_bytes / (vec16 ? 16 : 2);
  long long z = (2 * 148 + blocks - 1) / blocks;
  if (z > (vecs + 255) / 256) z = (vecs + 255) / 256;
  if (z < 1) z = 1;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.layers2 + 1, (unsigned)G, (unsigned)z);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = vec16 ? cudaLaunchKernelEx(&cfg, beam::beam_reorder_kernel<KM, uint4>, p)
                        : cudaLaunchKernelEx(&cfg, beam::beam_reorder_kernel<KM, uint16_t>, p);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_beam_reorder(void* pools, const int32_t* own_table, int32_t* block_table,
                                const int32_t* seq_lens, const int32_t* parents, int G, int K,
                                int layers, int Hkv, int d, int P, int max_pages, int num_pages,
                                int elem, int32_t* status, cudaStream_t stream) {
  beam::ReorderParams p;
  p.pools = (uint8_t*)pools; p.own_table = own_table; p.block_table = block_table;
  p.seq_lens = seq_lens; p.parents = parents; p.status = status;
  p.tok_bytes = d * elem;
  p.head_bytes = P * p.tok_bytes;
  p.page_bytes = (long long)Hkv * p.head_bytes;
  p.pool_bytes = (long long)num_pages * p.page_bytes;
  p.K = K; p.layers2 = 2 * layers; p.Hkv = Hkv; p.P = P; p.max_pages = max_pages;
  p.num_pages = num_pages;
  const bool vec16 = p.tok_bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(pools) & 15) == 0;
  if (K <= 4) return launch_reorder_k<4>(p, G, vec16, stream);
  if (K <= 8) return launch_reorder_k<8>(p, G, vec16, stream);
  if (K <= 16) return launch_reorder_k<16>(p, G, vec16, stream);
  return launch_reorder_k<32>(p, G, vec16, stream);
}

}  // namespace llmc
