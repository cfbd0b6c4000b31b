// Beam search over the paged cache: the selection of a step and the reordering after it.
//
// beam_select: for every prompt, the n best of
//     score[k, v] = beam_score[k] + (x[k, v] - lse(x[k, :]))
// over its K beams and the vocabulary, in descending order, ties to the lowest k * V + v.
// One launch and no global workspace: a thread-block cluster owns a prompt and cuts its
// K rows into tasks (row, split).  A task is one pass over its logits: every thread keeps
// a running maximum and sum of exponentials, and the maximum of each of its cells (32
// elements, more in long rows) in shared memory.  The order inside a row is that of its
// logits, which needs no log-sum-exp, so the n best can be found before it is known: at
// least n elements reach the n-th largest of the (pairs of) threads' maxima, and only the
// few cells that reach it are read again.  Ranks come from comparing all pairs of the few
// survivors (rows of very many equal logits go through sorted lists instead).  The cluster's first
// CTA fetches the tasks' lists and sums through distributed shared memory and ranks the
// candidates by their scores in the same way.
// Bound: the logits are read once from HBM; then the exponentials (16 a cycle and SM).
// Measured on 64 prompts of 8 beams, 131 MB of bf16 logits: 41 us captured and called (floor 20
// us), some 29 of them the stream; with lists kept up to date while streaming instead of cells
// 104 us.  A CTA's tasks run one after another: nothing streams while a row is ranked (8 prompts
// of 32 beams, two rows a CTA: 72 us, floor 10).
//
// Sums of exponentials are held in fp32 per thread, joined in fp32 inside a split and in
// fp64 across splits: a log-sum-exp is good to 2^-20.  Scores are ranked in
// fp64 (at -12 and less, candidates of different beams are often closer than fp32 tells apart)
// and rounded once to fp32.
//
// beam_reorder: beam i of a prompt continues from beam parent[i].  See below.
#include <climits>
#include <string>

#include "common.cuh"

namespace llmc {
namespace beam {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBeams = 32;   // five bits of a candidate's tie
constexpr int kU = 4;           // 16-byte vectors of a tile per lane; two more tiles in flight
constexpr int kCells = 32;      // cells of a thread

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
// values (0 and -0 too) rank by the lowest index.  Never zero for a number (0: "no entry").
__device__ __forceinline__ unsigned long long make_key(float f, uint32_t idx) {
  uint32_t u = __float_as_uint(f + 0.f);
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

// 2^x by the hardware (2 ulp); exp2f adds a range check for results below 2^-126, which
// a sum whose largest term is 1 does not notice.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations at once.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The words of a vector: elements per word, their values, the larger of two words by element.
template <typename T>
struct Word;
template <>
struct Word<float> {
  static constexpr int kN = 1;
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float top(uint32_t a) { return __uint_as_float(a); }
  static __device__ __forceinline__ float get(uint32_t a, int) { return __uint_as_float(a); }
};
template <>
struct Word<__half> {
  static constexpr int kN = 2;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float get(uint32_t a, int e) {
    return __half2float(__ushort_as_half((unsigned short)(e ? a >> 16 : a & 0xffffu)));
  }
  static __device__ __forceinline__ float top(uint32_t a) { return fmaxf(get(a, 0), get(a, 1)); }
};
template <>
struct Word<__nv_bfloat16> {
  static constexpr int kN = 2;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a),
                                     *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float get(uint32_t a, int e) {
    return __uint_as_float(e ? a & 0xffff0000u : a << 16);
  }
  static __device__ __forceinline__ float top(uint32_t a) { return fmaxf(get(a, 0), get(a, 1)); }
};

// Vectors of a row by index from the aligned ones that were fetched: vector v holds elements
// [v VEC, v VEC + VEC) of the row, the fetched ones begin h elements (0 < h < VEC) earlier.  The
// rest of a lane's vectors is in the next lane, the last lane's in the first lane's next one.
// Vectors from `left` on are -inf.
template <typename T>
__device__ __forceinline__ void realign(uint4 (&tile)[kU], const uint4& behind, int h, int lane,
                                        int left) {
  const int bytes = h * (int)sizeof(T);
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const uint4 a = tile[u], b = u + 1 < kU ? tile[u + 1 < kU ? u + 1 : u] : behind;
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[4 + i] = __shfl_sync(0xffffffffu, lane ? w[i] : w[4 + i], (lane + 1) & 31);
    if (bytes & 8)
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    if (bytes & 4)
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    if (bytes & 2)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __byte_perm(w[i], w[i + 1], 0x5432);
    constexpr uint32_t F = Word<T>::kNegInf;
    tile[u] = u * 32 + lane < left ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(F, F, F, F);
  }
}

// How many of the n descending entries of a are better than `key`.
__device__ __forceinline__ int count_better(const unsigned long long* a, int n,
                                            unsigned long long key) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] > key) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// Merges the warps' sorted lists (buf[w * kCap], len[w] entries) into the n best, in out;
// the rest of out is 0.  tmp: 6 * n keys, tlen: 6 lengths.  All threads of the block.
// In pairs: an element's rank is its place plus a binary search in the other list.
__device__ __noinline__ void merge_warps(const unsigned long long* buf, const int* len, int n,
                                         unsigned long long* tmp, int* tlen,
                                         unsigned long long* out) {
  const int tid = threadIdx.x;
  for (int i = tid; i < n; i += kThreads) out[i] = 0ull;
  __syncthreads();
  for (int level = 0; level < 3; ++level) {
    const int pairs = 4 >> level;
    // level 0: the warps' lists -> tmp[0..3], level 1: -> tmp[4..5], level 2: -> out
    const unsigned long long* src = level == 0 ? buf : level == 1 ? tmp : tmp + 4 * n;
    const int stride = level == 0 ? kCap : n;
    const int* sl = level == 0 ? len : level == 1 ? tlen : tlen + 4;
    unsigned long long* dst = level == 2 ? out : level == 0 ? tmp : tmp + 4 * n;
    for (int i = tid; i < pairs * 2 * n; i += kThreads) {
      const int w = i / n, j = i - w * n;       // list, place
      if (j >= sl[w]) continue;
      const unsigned long long key = src[w * stride + j];
      const int r = j + count_better(src + (w ^ 1) * stride, sl[w ^ 1], key);
      if (r < n) dst[(w >> 1) * n + r] = key;
    }
    if (level < 2 && tid < pairs)
      tlen[4 * level + tid] = min(n, sl[2 * tid] + sl[2 * tid + 1]);
    __syncthreads();
  }
}

// A candidate: its fp64 score as bits that order like it (0: no entry), and what decides
// between equal ones, the lower the better: beam, falling logit, token.  (Logits of a beam
// may differ by less than its scores can show; their order is that of the logits' lists,
// which is what merging these relies on.)
constexpr int kTokenBits = 27;
struct __align__(16) Cand {
  unsigned long long score, tie;
};
__device__ __forceinline__ unsigned long long make_tie(int beam, uint32_t logit, uint32_t token) {
  return (unsigned long long)beam << 59 | (unsigned long long)~logit << kTokenBits | token;
}
__device__ __forceinline__ unsigned long long score_bits(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);   // no -0
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double bits_score(unsigned long long u) {
  return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u));
}
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
  return a.score > b.score || (a.score == b.score && a.tie < b.tie);
}

// Candidates of the merge space: half the lists, or what all pairs are compared of.
__host__ __device__ inline int spare_cands(int n, int tasks) {
  const int halved = (tasks + 1) / 2 * n, most = tasks * n < kThreads ? tasks * n : kThreads;
  return halved > most ? halved : most;
}
// Bytes of dynamic shared memory (see the kernel).
__host__ __device__ inline size_t select_smem(int K, int n, int tasks, int per_cta) {
  const size_t keys = (size_t)kWarps * kCap + 6 * (size_t)n + (size_t)per_cta * (n + 1) +
                      (size_t)tasks * (n + 1) + (size_t)kCells * kThreads / 2;
  const size_t cands = (size_t)tasks * n + spare_cands(n, tasks);
  return (keys + (keys & 1)) * 8 + cands * sizeof(Cand) + (size_t)K * 24;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) beam_select_kernel(const SelectParams p) {
  constexpr int VEC = 16 / sizeof(T), WN = Word<T>::kN;
  extern __shared__ __align__(16) uint8_t sm_raw[];
  const int n = p.n, K = p.K, V = p.V, S = p.splits;
  const uint32_t rank = cluster_ctarank(), C = cluster_nctarank();
  const int g = blockIdx.x / C;
  const int tasks = K * S;
  const int per_cta = (tasks + (int)C - 1) / (int)C;
  // shared: warp buffers [kWarps][kCap], merge space [6][n], this CTA's lists [per_cta][n]
  // and sums [per_cta], cells [kCells][kThreads]; then (first CTA) all lists [tasks][n] and
  // sums, the candidates and their merge space, row constants.
  unsigned long long* wbuf = reinterpret_cast<unsigned long long*>(sm_raw);
  unsigned long long* tmp = wbuf + kWarps * kCap;
  unsigned long long* lists = tmp + 6 * n;
  unsigned long long* sums = lists + (size_t)per_cta * n;       // (max, sum) as two floats
  float* cells = reinterpret_cast<float*>(sums + per_cta);
  unsigned long long* all = sums + per_cta + kCells * kThreads / 2;
  unsigned long long* all_sums = all + (size_t)tasks * n;
  const size_t keys = (size_t)kWarps * kCap + 6 * n + (size_t)per_cta * (n + 1) +
                      (size_t)tasks * (n + 1) + kCells * kThreads / 2;
  Cand* cand = reinterpret_cast<Cand*>(wbuf + keys + (keys & 1));
  Cand* half = cand + (size_t)tasks * n;
  // of a row: log-sum-exp = row_max + row_log, beam score, 0 live, 1 dead, 2 finished
  double* row_log = reinterpret_cast<double*>(half + spare_cands(n, tasks));
  double* row_b = row_log + K;
  float* row_max = reinterpret_cast<float*>(row_b + K);
  int* row_kind = reinterpret_cast<int*>(row_max + K);
  __shared__ float red_m[kWarps], red_s[kWarps], red_b[kWarps];
  __shared__ __align__(16) float maxima[kThreads / 2];
  __shared__ int hits[kThreads];
  __shared__ int wcount[kWarps], tlen[6], n_hits, survivors;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();

  constexpr float kLog2e = 1.4426950408889634f;
  const float kNegInf = __int_as_float(0xff800000);
  const uint64_t l2e = pair(kLog2e, kLog2e);

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
    // A row is cut by the index of its elements, wherever it begins: vector v holds elements
    // [v VEC, v VEC + VEC).  Rows of equal logits so have the same sums, bit for bit, and tie.
    // A row that begins h elements behind a 16-byte boundary is fetched from that boundary on
    // and its vectors are put together from two neighbours (see realign; 64 prompts of 8 beams,
    // V 128255: 48.7 us, cut by address, which ties of rows at odd strides do not survive, 41.7).
    const int h = (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % VEC);
    const int nvec = (V + VEC - 1) / VEC;
    const int v0 = (int)((long long)nvec * split / S), v1 = (int)((long long)nvec * (split + 1) / S);
    // A warp's vectors are contiguous, so its later elements have larger indices.
    const int w0 = v0 + (int)((long long)(v1 - v0) * warp / kWarps);
    const int w1 = v0 + (int)((long long)(v1 - v0) * (warp + 1) / kWarps);
    // Fetched vectors that are whole: [whole0, whole1).
    const uint4* vec = reinterpret_cast<const uint4*>(x - h) + lane;
    const int last = h ? w1 + 1 : w1, whole0 = h ? 1 : 0, whole1 = min(last, (V + h) / VEC);
    auto load = [&](int base, uint4 (&raw)[kU]) {
      if (base >= whole0 && base + 32 * kU <= whole1) {
#pragma unroll
        for (int u = 0; u < kU; ++u) raw[u] = __ldg(vec + base + u * 32);
        return;
      }
      // the ends of a row, or past this warp's part: -inf outside
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int v = base + u * 32 + lane;
        const long long e0 = (long long)v * VEC - h;
        constexpr uint32_t F = Word<T>::kNegInf;
        raw[u] = make_uint4(F, F, F, F);
        if (v >= last) continue;
        if (v >= whole0 && v < whole1) {
          raw[u] = __ldg(vec + base + u * 32);
        } else {
          T* r = reinterpret_cast<T*>(&raw[u]);
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (e0 + e >= 0 && e0 + e < V) r[e] = x[e0 + e];
        }
      }
    };
    // One pass: maximum, sum, cells.
    float m = kNegInf, ref = 0.f;    // ref = m; 0 while m = -inf
    uint64_t s2 = pair(0.f, 0.f);
    // tiles of a cell, the same for all warps
    const int tiles = ((v1 - v0 + kWarps - 1) / kWarps + 32 * kU - 1) / (32 * kU);
    const int per_cell = (tiles + kCells - 1) / kCells;
    float cell_m = kNegInf;
    int in_cell = 0, cell = 0;
    uint4 cur[kU], ahead[kU];
    load(w0, cur);
    load(w0 + 32 * kU, ahead);
    for (int base = w0; base < w1; base += 32 * kU) {
      uint4 next[kU];
      load(base + 64 * kU, next);
      if (h) realign<T>(cur, ahead[0], h, lane, w1 - base);
      const uint32_t* wd = reinterpret_cast<const uint32_t*>(cur);
      uint32_t mw = wd[0];
#pragma unroll
      for (int i = 1; i < kU * 4; ++i) mw = Word<T>::max(mw, wd[i]);
      const float tile_m = Word<T>::top(mw);
      cell_m = fmaxf(cell_m, tile_m);
      if (++in_cell == per_cell || base + 32 * kU >= w1) {
        cells[cell * kThreads + threadIdx.x] = cell_m;
        cell_m = kNegInf;
        in_cell = 0;
        ++cell;
      }
      // Exponents are (x - m) log2(e), the difference first: never positive, and 0 at the
      // maximum, for logits of any size (finite masks up to the type's lowest value).
      if (tile_m > m) {
        const float f = ex2((m - tile_m) * kLog2e);
        const float2 o = unpair(s2);
        s2 = pair(o.x * f, o.y * f);
        m = ref = tile_m;
      }
      const uint64_t nref = pair(-ref, -ref);
#pragma unroll
      for (int i = 0; i < kU * 4; i += 3 - WN) {
        const float a = Word<T>::get(wd[i], 0);
        const float b = WN == 2 ? Word<T>::get(wd[i], 1) : Word<T>::get(wd[i + 1], 0);
        const float2 e = unpair(mul2(add2(pair(a, b), nref), l2e));
        s2 = add2(s2, pair(ex2(e.x), ex2(e.y)));
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        cur[u] = ahead[u];
        ahead[u] = next[u];
      }
    }
    // Join the maxima and sums, and the bound on the n-th best.
    const float2 sp = unpair(s2);
    float s = sp.x + sp.y;               // NaN: a NaN, or an infinity, among the logits
    float wm = m;
    for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
    float ws = m == kNegInf ? s : s * ex2((m - wm) * kLog2e);
    for (int o = 16; o; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
    const float m2 = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));   // of two threads
    if (!(lane & 1)) maxima[threadIdx.x >> 1] = m2;
    if (lane == 0) {
      red_m[warp] = wm;
      red_s[warp] = ws;
    }
    if (threadIdx.x == 0) n_hits = survivors = 0;
    __syncthreads();
    // The n-th largest of the maxima of two threads: the least of those that fewer than n
    // exceed.  Each of the two counts in one half.
    int above = 0;
#pragma unroll 4
    for (int i = (lane & 1) * (kThreads / 4), e = i + kThreads / 4; i < e; i += 4) {
      const float4 o = *reinterpret_cast<const float4*>(maxima + i);
      above += (o.x > m2) + (o.y > m2) + (o.z > m2) + (o.w > m2);
    }
    above += __shfl_xor_sync(0xffffffffu, above, 1);
    float wb = above < n ? m2 : __int_as_float(0x7f800000);
    for (int o = 16; o; o >>= 1) wb = fminf(wb, __shfl_xor_sync(0xffffffffu, wb, o));
    if (lane == 0) red_b[warp] = wb;
    if (threadIdx.x == 0) {
      float M = kNegInf;
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, red_m[w]);
      float sum = 0.f;
      for (int w = 0; w < kWarps; ++w)
        sum += red_m[w] == kNegInf ? red_s[w] : red_s[w] * ex2((red_m[w] - M) * kLog2e);
      sums[slot] = ((unsigned long long)__float_as_uint(M) << 32) | __float_as_uint(sum);
    }
    __syncthreads();
    float bound = red_b[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) bound = fminf(bound, red_b[w]);
    for (int i = threadIdx.x; i < n; i += kThreads) out[i] = 0ull;
    for (int c = 0; c < cell; ++c)
      if (cells[c * kThreads + threadIdx.x] >= bound) {
        const int at = atomicAdd(&n_hits, 1);
        if (at < kThreads) hits[at] = c << 8 | (int)threadIdx.x;
      }
    __syncthreads();
    const int hit_n = n_hits;
    if (hit_n <= kThreads) {
      // A warp per cell, a lane per element.
#pragma unroll 2
      for (int i = warp; i < hit_n; i += kWarps) {
        const int c = hits[i] >> 8, th = hits[i] & 255, tw = th >> 5;
        const int tw0 = v0 + (int)((long long)(v1 - v0) * tw / kWarps);
        const int tw1 = v0 + (int)((long long)(v1 - v0) * (tw + 1) / kWarps);
        for (int b = 0; b < per_cell; ++b) {
          const int u = lane / VEC, v = tw0 + (c * per_cell + b) * 32 * kU + u * 32 + (th & 31);
          const long long idx = (long long)v * VEC + lane % VEC;
          float f = kNegInf;
          const bool in = lane < kU * VEC && v < tw1 && idx < V;
          if (in) f = to_f32(x[idx]);
          const bool pass = in && f >= bound;
          const unsigned vote = __ballot_sync(0xffffffffu, pass);
          if (!vote) continue;
          int at = 0;
          if (lane == 0) at = atomicAdd(&survivors, __popc(vote));
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(vote & ((1u << lane) - 1u));
          if (pass && at < kThreads) wbuf[at] = make_key(f, (uint32_t)idx);
        }
      }
    }
    __syncthreads();
    if (hit_n <= kThreads && survivors <= kThreads) {   // all pairs: a thread ranks one survivor
      const int total = survivors;
      if ((int)threadIdx.x < total) {
        const unsigned long long key = wbuf[threadIdx.x];
        int r = 0;
#pragma unroll 4
        for (int i = 0; i < total; ++i) r += wbuf[i] > key ? 1 : 0;
        if (r < n) out[r] = key;
      }
      __syncthreads();
      continue;
    }
    // Very many equal logits: sorted lists.
    // Read the cells that reach the bound again, in the order of their indices.
    WarpTop top;
    top.buf = wbuf + warp * kCap;
    top.n = n;
    top.count = 0;
    top.tau = kNegInf;
    top.full = false;
    for (int c = 0; c < cell; ++c) {
      const float cm = cells[c * kThreads + threadIdx.x];
      if (!__any_sync(0xffffffffu, cm >= bound && (!top.full || cm > top.tau))) continue;
      const int end = min(w1, w0 + (c + 1) * per_cell * 32 * kU);
      for (int base = w0 + c * per_cell * 32 * kU; base < end; base += 32 * kU) {
        uint4 raw[kU];
        if (h == 0) {
          load(base, raw);
        } else {
          T* r = reinterpret_cast<T*>(raw);
#pragma unroll
          for (int i = 0; i < kU * VEC; ++i) {
            const long long idx = (long long)(base + i / VEC * 32 + lane) * VEC + i % VEC;
            constexpr uint32_t F = Word<T>::kNegInf;
            r[i] = idx < V ? x[idx] : *reinterpret_cast<const T*>(&F);
          }
        }
        const uint32_t* wd = reinterpret_cast<const uint32_t*>(raw);
        const bool strict = top.full && top.tau >= bound;
        const float lo = top.full ? fmaxf(top.tau, bound) : bound;
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < kU * VEC; ++i) {
          const float f = Word<T>::get(wd[i / WN], i % WN);
          mask |= (strict ? f > lo : f >= lo) ? 1u << i : 0u;
        }
        while (true) {
          bool pass = mask != 0;
          if (!__any_sync(0xffffffffu, pass)) break;
          const int bit = pass ? __ffs(mask) - 1 : 0;
          mask &= mask - 1;
          const int v = base + (bit / VEC) * 32 + lane;
          const long long idx = (long long)v * VEC + bit % VEC;
          pass = pass && v < w1 && idx < V;
          const float f = pass ? to_f32(x[idx]) : 0.f;
          unsigned vote = __ballot_sync(0xffffffffu, pass);
          if (top.count + __popc(vote) > kCap) {
            // Elements of this tile are in no order: equal values still compete by index.
            top_compact(top, lane);
            pass = pass && (!top.full || f >= top.tau);
            vote = __ballot_sync(0xffffffffu, pass);
          }
          if (pass)
            top.buf[top.count + __popc(vote & ((1u << lane) - 1u))] = make_key(f, (uint32_t)idx);
          top.count += __popc(vote);
        }
      }
    }
    top_compact(top, lane);
    if (lane == 0) wcount[warp] = top.count;
    __syncthreads();
    merge_warps(wbuf, wcount, n, tmp, tlen, out);
  }
  cluster_sync_all();   // every list is written
  if (rank == 0) {      // all lists and sums, from the CTA that made them
    for (int i = threadIdx.x; i < tasks * (n + 1); i += kThreads) {
      const int t = i / (n + 1), j = i - t * (n + 1);
      const unsigned long long* from = j < n ? lists + (size_t)(t / (int)C) * n + j : sums + t / (int)C;
      const unsigned long long v = ld_dsmem_u64(dsmem_addr(smem_u32(from), (uint32_t)(t % (int)C)));
      if (j < n) all[(size_t)t * n + j] = v; else all_sums[t] = v;
    }
  }
  cluster_sync_all();   // the peers' shared memory has been read
  if (rank != 0) return;
  for (int k = threadIdx.x; k < K; k += kThreads) {
    const long long gk = (long long)g * K + k;
    const float b = p.beam_scores[gk];
    float M = kNegInf;
    double sum = 0.0;
    for (int sp = 0; sp < S; ++sp)
      M = fmaxf(M, __uint_as_float((uint32_t)(all_sums[k * S + sp] >> 32)));
    for (int sp = 0; sp < S; ++sp) {
      const unsigned long long u = all_sums[k * S + sp];
      const float mt = __uint_as_float((uint32_t)(u >> 32)), st = __uint_as_float((uint32_t)u);
      sum += mt == kNegInf ? st : (double)(st * ex2((mt - M) * kLog2e));
    }
    const double lg = log(sum);
    const bool fin = p.finished && p.finished[gk];
    row_b[k] = (double)b;
    row_log[k] = lg;
    row_max[k] = M;
    row_kind[k] = !isfinite(b) ? 1 : fin ? 2 : isfinite(M) && isfinite(lg) ? 0 : 1;
  }
  if (threadIdx.x == 0) survivors = 0;
  __syncthreads();
  // The candidates.  Rows without usable scores offer their lowest tokens at -inf, finished
  // rows eos and then those; both in their first list.
  for (int i = threadIdx.x; i < tasks * n; i += kThreads) {
    const int t = i / n, j = i - t * n, k = t / S;
    Cand c;
    double sc = -INFINITY;
    c.score = 0ull;                      // no entry
    c.tie = i;
    const int kind = row_kind[k];
    if (kind == 0) {
      const unsigned long long key = all[i];
      if (key != 0ull) {
        sc = row_b[k] + (((double)key_value(key) - (double)row_max[k]) - row_log[k]);
        c.score = score_bits(sc);
        c.tie = make_tie(k, (uint32_t)(key >> 32), key_index(key));
      }
    } else if (t == k * S) {
      int tok = j;
      if (kind == 2) {
        tok = j == 0 ? p.eos : j - 1 < p.eos ? j - 1 : j;
        if (j == 0) sc = row_b[k];
      }
      if (tok < V) {
        c.score = score_bits(sc);
        c.tie = make_tie(k, 0u, (uint32_t)tok);
      }
    }
    cand[i] = c;
  }
  __syncthreads();
  // Every list has n entries, so the best of their last ones bounds the n-th best.
  unsigned long long bound = 0;
#pragma unroll 4
  for (int t = 0; t < tasks; ++t) {
    const unsigned long long o = cand[(size_t)t * n + n - 1].score;
    bound = o > bound ? o : bound;
  }
  for (int i = threadIdx.x; i < tasks * n; i += kThreads)
    if (cand[i].score >= bound) {
      const int at = atomicAdd(&survivors, 1);
      if (at < kThreads) half[at] = cand[i];
    }
  __syncthreads();
  Cand* src = cand;
  if (survivors <= kThreads) {
    // Eight lanes compare a survivor with all others.
    const int total = survivors;
    for (int i = threadIdx.x >> 3; i < (total + 3) / 4 * 4; i += kThreads / 8) {
      const Cand c = half[min(i, total - 1)];
      int r = 0;
#pragma unroll 2
      for (int o = lane & 7; o < total; o += 8) r += better(half[o], c) ? 1 : 0;
      r += __shfl_xor_sync(0xffffffffu, r, 1);
      r += __shfl_xor_sync(0xffffffffu, r, 2);
      r += __shfl_xor_sync(0xffffffffu, r, 4);
      if ((lane & 7) == 0 && i < total && r < n) cand[r] = c;
    }
    __syncthreads();
  } else {
    // Merge the tasks' lists in pairs until one is left.
    Cand* dst = half;
    for (int left = tasks; left > 1; left = (left + 1) / 2) {
      for (int i = threadIdx.x; i < left * n; i += kThreads) {
        const int w = i / n, j = i - w * n;
        const Cand c = src[i];
        int r = j;
        if ((w ^ 1) < left) {
          const Cand* o = src + (size_t)(w ^ 1) * n;
          int lo = 0, hi = n;
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (better(o[mid], c)) lo = mid + 1; else hi = mid;
          }
          r += lo;
        }
        if (r < n) dst[(size_t)(w >> 1) * n + r] = c;
      }
      __syncthreads();
      Cand* x = src;
      src = dst;
      dst = x;
    }
  }
  for (int r = threadIdx.x; r < n; r += kThreads) {
    const long long o = (long long)g * n + r;
    const Cand c = src[r];
    p.out_scores[o] = (float)bits_score(c.score);
    p.out_beams[o] = (int32_t)(c.tie >> 59);
    p.out_tokens[o] = (int64_t)(c.tie & ((1ull << kTokenBits) - 1));
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
// table is moved the same way, a thread per column.  Bound: HBM (the moved tokens; 113 us for
// 638 MB, 86% of a plain copy's rate), and at small sizes the launch (2.9 us captured, 9.3 us
// from the host).
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
  // CTAs per prompt: as many as run at once, two per SM (64 prompts of 8 beams: 4 CTAs each
  // 41 us, 8 CTAs 44 to 52 us, 16 CTAs 63 us: what a row costs besides its logits).
  int C = 16;
  while (C > 1 && (long long)G * C > 2 * 148) C /= 2;
  p.splits = C / p.K > 1 ? C / p.K : 1;
  const int tasks = p.K * p.splits, per = (tasks + C - 1) / C;
  const size_t smem = beam::select_smem(p.K, p.n, tasks, per);
  cudaError_t e = allow_shared_memory<beam::beam_select_kernel<T>>(true);
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
