// Single-token decode attention for a batch whose sequences share prefixes, paged K/V.
//
//   out[b, h] = softmax_t(q[b, h] . k_t * scale) . v_t   over the seq_lens[b] tokens of b
//
// For a group of n sequences with a common prefix of s tokens, the n * R query rows that
// use one KV head (R = query heads per KV head) meet the same s keys and values: one
// matrix product that reads them once, where separate sequences read them n times.  The
// tokens behind the prefix are a sequence's own.  Both parts leave a normalised partial
// and its log2-sum-exp per row, and the parts are joined by
//   M = max lse_i,  out = sum 2^(lse_i - M) o_i / sum 2^(lse_i - M).
// Scores, maxima, sums and partials are fp32; only out is rounded to the tensor type.
//
// bf16/fp16 at head size 64 or 128 and pages of 8, 16, 32, 64 or a multiple of 128 tokens
// run on the tensor cores (shared_prefix_tc.cuh).  The kernels of this file take every
// other type, head size and page size: shared-prefix rows and own rows alike are cut into
// units of 16 or 64 query rows x a range of tokens, in fp32 on the CUDA cores, with 32
// tokens of K and V at a time in shared memory.  Bound: the FMA pipes and, as evenly, the
// shared-memory reads that feed them (4 rows x 2 tokens or 4 rows x 4 columns a thread).
// Measured in fp32: 24 us for 1.7 MB (launches and dependent loads), 230 us for 408 MB of K and
// V with 4 query rows per KV head (1.8 TB/s).
#include <climits>
#include <string>

#include "shared_prefix_tc.cuh"

namespace llmc {
namespace prefix {
namespace generic {

constexpr int kTok = 32;      // tokens per step
constexpr int kThreads = 256; // 16 threads per group of rows

// Shared memory of a unit of 16 * RPT rows: Q, K (rows of dp + 4 floats), V, P.
__host__ __device__ inline size_t smem_floats(int rpt, int dp) {
  return (size_t)16 * rpt * (dp + 4) + (size_t)kTok * (dp + 4) + (size_t)kTok * dp +
         (size_t)16 * rpt * (kTok + 4);
}

// Where a block works.
struct Unit {
  int lo, nrows, row0, table_row, hk, first, last, slot;
  bool group;
};

// Attention of rows [row0, row0 + 16 RPT) over tokens [first, last).  Thread (rg, c): rows
// rg * RPT ..., keys c and c + 16, output columns 4 c + 64 j.
template <typename T, int NJ, int RPT>
__device__ __forceinline__ void attend(const Params& p, const Unit& u, float* sm) {
  constexpr int DP = 64 * NJ, QS = DP + 4, PS = kTok + 4, ROWS = 16 * RPT;
  float* Qs = sm;                 // [ROWS][QS]
  float* Ks = Qs + ROWS * QS;     // [32][QS]
  float* Vs = Ks + kTok * QS;     // [32][DP]
  float* Ps = Vs + kTok * DP;     // [ROWS][PS]
  const int d = p.d, tid = threadIdx.x, rg = tid >> 4, c = tid & 15;
  const T* q = reinterpret_cast<const T*>(p.q);
  for (int i = u.first < u.last ? tid : ROWS * DP; i < ROWS * DP; i += kThreads) {
    const int r = i / DP, col = i - r * DP, row = u.row0 + r;
    float v = 0.f;
    if (row < u.nrows && col < d) {
      const int b = u.lo + row / p.R, h = u.hk * p.R + row % p.R;
      v = to_f32(q[((long long)b * p.Hq + h) * d + col]) * p.scale_log2;
    }
    Qs[r * QS + col] = v;
  }
  const T* kp = reinterpret_cast<const T*>(p.k_pages);
  const T* vp = reinterpret_cast<const T*>(p.v_pages);
  constexpr int VEC = 16 / sizeof(T);
  const bool vec = d % VEC == 0 && ((reinterpret_cast<uintptr_t>(kp) |
                                     reinterpret_cast<uintptr_t>(vp)) & 15) == 0;
  const float kNegInf = __int_as_float(0xff800000);
  float m[RPT], l[RPT], acc[RPT][NJ][4];
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    m[r] = kNegInf;
    l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r][j][e] = 0.f;
  }
  // 8 threads per token bring its key and value; columns from d on are zero.  A step's vectors
  // are on their way while the step before is computed, its page numbers a step earlier still
  // (10 sequences of up to 25000 tokens at 4 fp32 KV heads of 64: 234 us, fetched when needed
  // 259 us; 383 us when warps without a row computed too).
  constexpr int NV = DP / (8 * VEC);
  constexpr bool kAhead = RPT == 1 && NV <= 4;  // beyond that the registers cost more
  const int t = tid >> 3, part = tid & 7;
  uint4 kr[NV], vr[NV];
  const int32_t* table = p.block_table + (long long)u.table_row * p.max_pages;
  auto page_at = [&](int t0) { return t0 + t < u.last ? table[(t0 + t) / p.P] : 0; };
  auto offset = [&](int t0, int page) -> long long {
    if (page < 0 || page >= p.num_pages) {
      atomicOr(p.status, kStatusBadPage);
      page = 0;
    }
    return (((long long)page * p.Hkv + u.hk) * p.P + (t0 + t) % p.P) * d;
  };
  auto fetch = [&](int t0, int page) {
    const bool have = t0 + t < u.last;
    const long long base = have ? offset(t0, page) : 0;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = (part + 8 * n) * VEC;
      const bool in = have && i < d;
      kr[n] = in ? __ldg(reinterpret_cast<const uint4*>(kp + base + i)) : make_uint4(0u, 0u, 0u, 0u);
      vr[n] = in ? __ldg(reinterpret_cast<const uint4*>(vp + base + i)) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  const bool live = u.row0 + (tid >> 5) * 2 * RPT < u.nrows;   // does this warp have a row?
  int page = page_at(u.first);
  if (vec && kAhead) {
    fetch(u.first, page);
    page = page_at(u.first + kTok);
  }
  for (int t0 = u.first; t0 < u.last; t0 += kTok) {
    const int nt = min(kTok, u.last - t0);
    __syncthreads();
    if (vec) {
      if (!kAhead) fetch(t0, page);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int i = (part + 8 * n) * VEC;
        const T* ke = reinterpret_cast<const T*>(&kr[n]);
        const T* ve = reinterpret_cast<const T*>(&vr[n]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          Ks[t * QS + i + e] = to_f32(ke[e]);
          Vs[t * DP + i + e] = to_f32(ve[e]);
        }
      }
    } else {
      const bool have = t < nt;
      const long long base = have ? offset(t0, page) : 0;
      for (int i = part; i < DP; i += 8) {
        const bool in = have && i < d;
        Ks[t * QS + i] = in ? to_f32(kp[base + i]) : 0.f;
        Vs[t * DP + i] = in ? to_f32(vp[base + i]) : 0.f;
      }
    }
    __syncthreads();
    if (vec && kAhead) {
      fetch(t0 + kTok, page);
      page = page_at(t0 + 2 * kTok);
    } else {
      page = page_at(t0 + kTok);
    }
    if (!live) continue;
    float x0[RPT], x1[RPT];
#pragma unroll
    for (int r = 0; r < RPT; ++r) x0[r] = x1[r] = 0.f;
#pragma unroll 4
    for (int i = 0; i < DP; i += 4) {
      const float4 k0 = *reinterpret_cast<const float4*>(Ks + c * QS + i);
      const float4 k1 = *reinterpret_cast<const float4*>(Ks + (c + 16) * QS + i);
#pragma unroll
      for (int r = 0; r < RPT; ++r) {
        const float4 qv = *reinterpret_cast<const float4*>(Qs + (rg * RPT + r) * QS + i);
        x0[r] = fmaf(qv.x, k0.x, fmaf(qv.y, k0.y, fmaf(qv.z, k0.z, fmaf(qv.w, k0.w, x0[r]))));
        x1[r] = fmaf(qv.x, k1.x, fmaf(qv.y, k1.y, fmaf(qv.z, k1.z, fmaf(qv.w, k1.w, x1[r]))));
      }
    }
#pragma unroll
    for (int r = 0; r < RPT; ++r) {
      if (c >= nt) x0[r] = kNegInf;
      if (c + 16 >= nt) x1[r] = kNegInf;
      float tm = fmaxf(x0[r], x1[r]);
#pragma unroll
      for (int o = 8; o; o >>= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, o));
      const float mn = fmaxf(m[r], tm);
      const float mu = mn == kNegInf ? 0.f : mn;    // every score -inf: weights 0
      const float f = exp2f(m[r] - mu);
      const float p0 = exp2f(x0[r] - mu), p1 = exp2f(x1[r] - mu);
      float ps = p0 + p1;
#pragma unroll
      for (int o = 8; o; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
      l[r] = l[r] * f + ps;
      m[r] = mn;
      Ps[(rg * RPT + r) * PS + c] = p0;
      Ps[(rg * RPT + r) * PS + c + 16] = p1;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][j][e] *= f;
    }
    __syncwarp();                                 // a row's threads are in one warp
    // Weights behind nt are zero and so are V's rows there.
#pragma unroll 2
    for (int t = 0; t < kTok; t += 4) {
      if (t >= nt) break;
      float4 w[RPT];
#pragma unroll
      for (int r = 0; r < RPT; ++r)
        w[r] = *reinterpret_cast<const float4*>(Ps + (rg * RPT + r) * PS + t);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const float4 v = *reinterpret_cast<const float4*>(Vs + (t + e) * DP + 64 * j + 4 * c);
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            const float pw = e == 0 ? w[r].x : e == 1 ? w[r].y : e == 2 ? w[r].z : w[r].w;
            acc[r][j][0] = fmaf(pw, v.x, acc[r][j][0]);
            acc[r][j][1] = fmaf(pw, v.y, acc[r][j][1]);
            acc[r][j][2] = fmaf(pw, v.z, acc[r][j][2]);
            acc[r][j][3] = fmaf(pw, v.w, acc[r][j][3]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RPT; ++r) {
    const int row = u.row0 + rg * RPT + r;
    if (row >= u.nrows) continue;
    const int b = u.lo + row / p.R, h = u.hk * p.R + row % p.R;
    const long long o = ((long long)u.slot * p.B + b) * p.Hq + h;
    // An empty sequence has no part in its group's prefix.
    const bool none = l[r] == 0.f || (u.group && p.seq_lens[b] <= 0);
    const float inv = none ? 0.f : 1.f / l[r];
    if (!none) {                                 // an empty part's O is not read
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (64 * j + 4 * c + e < d) p.part_o[o * d + 64 * j + 4 * c + e] = acc[r][j][e] * inv;
    }
    if (c == 0) p.part_lse[o] = none ? kNegInf : m[r] + log2f(l[r]);
  }
}

// What the blocks have to know of the groups, once for all of them: groups[g] = {first
// sequence, end, shared tokens, leader (-1: all empty)}, and the shared tokens of every
// sequence.  One block: a warp per group.  (16 groups of 48 rows x 130 fp32 tokens: 68.0 us,
// with every block of units_kernel finding out for itself 70.6; the smallest case 24.0, 24.8.)
__global__ void __launch_bounds__(1024) groups_kernel(const Params p, int4* groups, int* seq_s) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  // One bad range and nothing is shared: the ranges may overlap.
  int bad = 0;
  for (int g = threadIdx.x; g < p.G; g += blockDim.x) {
    const int lo = p.starts[g], hi = p.starts[g + 1];
    bad |= lo < 0 || hi < lo || hi > p.B;
  }
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) seq_s[b] = 0;
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0) atomicOr(p.status, kStatusBadGroup);
  for (int g = threadIdx.x >> 5; g < p.G; g += blockDim.x >> 5) {
    const int lo = bad ? 0 : p.starts[g];
    const int hi = bad ? 0 : min(p.starts[g + 1], lo + min(p.max_group, p.B - lo));
    int mn = INT_MAX, first = INT_MAX;
    for (int b = lo + lane; b < hi; b += 32) {
      const int n = seq_len(p, b, false);
      if (n > 0) {
        mn = min(mn, n);
        first = min(first, b);
      }
    }
    mn = __reduce_min_sync(0xffffffffu, mn);
    first = __reduce_min_sync(0xffffffffu, first);
    const int s = first == INT_MAX ? 0 : max(0, min(p.shared[g], mn));
    if (lane == 0) groups[g] = make_int4(lo, hi, s, first == INT_MAX ? -1 : first);
    if (s)
      for (int b = lo + lane; b < hi; b += 32) seq_s[b] = s;
  }
}

// Partials: part_o [split_g + split_o][B * Hq][d], part_lse [split_g + split_o][B * Hq];
// slots below split_g are the shared part's, the others the own part's.
// Grid: x = unit of a KV head and split, y = KV head.  Units: the tiles of the groups' rows
// (16 * rpt rows; sized for max_group), then the 16-row tiles of every sequence.
// Three blocks per SM, for a few spilled words, up to head size 128 (16 groups of 48 rows x 130
// tokens at 8 fp32 KV heads of 128: 70.6 us, with two, as the compiler leaves it, 77.3 us).
template <typename T, int NJ>
__global__ void __launch_bounds__(kThreads, NJ <= 2 ? 3 : 1) units_kernel(
    const Params p, const int4* groups, const int* seq_s, int group_tiles, int seq_tiles, int rpt) {
  extern __shared__ __align__(16) float sm[];
  const int of_groups = p.G * group_tiles * p.split_g;
  Unit u;
  u.hk = blockIdx.y;
  u.group = (int)blockIdx.x < of_groups;
  const int splits = u.group ? p.split_g : p.split_o;
  const int unit = ((int)blockIdx.x - (u.group ? 0 : of_groups)) / splits;
  const int split = ((int)blockIdx.x - (u.group ? 0 : of_groups)) % splits;
  pdl_launch_dependents();
  pdl_wait();

  int t_begin, t_end;
  if (u.group) {
    const int4 g = groups[unit / group_tiles];
    u.lo = g.x;
    u.row0 = unit % group_tiles * 16 * rpt;
    u.nrows = (g.y - g.x) * p.R;
    // without shared tokens the sequences' own units mark the shared slots empty
    if (u.row0 >= u.nrows || g.z == 0) return;
    t_begin = 0;
    t_end = g.z;
    u.table_row = g.w;
  } else {
    u.lo = unit / seq_tiles;
    u.row0 = (unit % seq_tiles) * 16;
    u.nrows = p.R;
    t_end = seq_len(p, u.lo, split == 0 && threadIdx.x == 0);
    t_begin = min(seq_s[u.lo], t_end);
    u.table_row = u.lo;
    if (t_begin == 0 && split == 0)   // no shared part
      for (int i = threadIdx.x; i < 16 * p.split_g; i += kThreads)
        if (u.row0 + (i & 15) < u.nrows)
          p.part_lse[((long long)(i >> 4) * p.B + u.lo) * p.Hq + u.hk * p.R + u.row0 + (i & 15)] =
              __int_as_float(0xff800000);
  }
  // this block's share of the tokens, in whole steps
  const int steps = (t_end - t_begin + kTok - 1) / kTok;
  const int s0 = (int)((long long)steps * split / splits);
  const int s1 = (int)((long long)steps * (split + 1) / splits);
  u.first = t_begin + s0 * kTok;
  u.last = min(t_end, t_begin + s1 * kTok);
  u.slot = (u.group ? 0 : p.split_g) + split;
  if (u.group && rpt == 4)
    attend<T, NJ, 4>(p, u, sm);
  else
    attend<T, NJ, 1>(p, u, sm);
}

// One warp per row (b, h).
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
  pdl_launch_dependents();
  pdl_wait();
  const long long rows = (long long)p.B * p.Hq;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int n = p.split_g + p.split_o;
  float M = __int_as_float(0xff800000);
  for (int i = 0; i < n; ++i) M = fmaxf(M, p.part_lse[i * rows + row]);
  float acc[8], L = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  for (int i = 0; i < n; ++i) {
    const float lse = p.part_lse[i * rows + row];
    if (lse == __int_as_float(0xff800000)) continue;   // nothing in this part
    const float w = exp2f(lse - M);
    L += w;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane + 32 * j < p.d)
        acc[j] = fmaf(w, p.part_o[(i * rows + row) * p.d + lane + 32 * j], acc[j]);
  }
  T* out = reinterpret_cast<T*>(p.out) + row * p.d;
  const float inv = L > 0.f ? 1.f / L : L != L ? L : 0.f;   // an empty sequence gives zeros
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (lane + 32 * j < p.d) out[lane + 32 * j] = from_f32<T>(acc[j] * inv);
}

}  // namespace generic
}  // namespace prefix

namespace {
struct Device {
  int sms = 0, smem = 0;
};
Device device() {
  Device d;
  int dev = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
  cudaDeviceGetAttribute(&d.smem, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
  if (d.sms <= 0) d.sms = 148;   // no device (sizes are asked for on the host): a B200
  return d;
}

// Rows per thread of a group's units: 4 (64-row tiles) from 48 rows on, where a smaller tile
// would read K and V more often than a larger one wastes rows.
int generic_rpt(int Hq, int Hkv, int max_group) {
  return (long long)max_group * (Hq / Hkv) >= 48 ? 4 : 1;
}

// Splits of `units` units' tokens: enough blocks for four per SM, at most 16.
int generic_splits(long long units) {
  const long long s = (4 * 148 + units - 1) / (units > 0 ? units : 1);
  return (int)(s < 1 ? 1 : s > 16 ? 16 : s);
}
struct GenericPlan {
  int rpt, group_tiles, seq_tiles, split_g, split_o;
};
GenericPlan generic_plan(int B, int Hq, int Hkv, int G, int max_group) {
  GenericPlan z;
  const int R = Hq / Hkv;
  z.rpt = generic_rpt(Hq, Hkv, max_group);
  z.group_tiles = (int)(((long long)max_group * R + 16 * z.rpt - 1) / (16 * z.rpt));
  z.seq_tiles = (R + 15) / 16;
  z.split_g = G ? generic_splits((long long)Hkv * G * z.group_tiles) : 1;
  z.split_o = generic_splits((long long)Hkv * B * z.seq_tiles);
  return z;
}

size_t generic_tables(int B, int G) {   // groups_kernel's, in front of the partials
  return ((size_t)G * sizeof(int4) + (size_t)B * sizeof(int) + 15) / 16 * 16;
}

size_t generic_workspace(int B, int Hq, int Hkv, int d, int G, int max_group) {
  const GenericPlan z = generic_plan(B, Hq, Hkv, G, max_group);
  return (size_t)(z.split_g + z.split_o) * B * Hq * ((size_t)d + 1) * sizeof(float) +
         generic_tables(B, G);
}

// Workspace of the tensor-core kernels: plan, tables (if they do not fit shared memory),
// partials of shared and of own units.
struct TcSizes {
  size_t plan, tables, o, lse, own_o, own_lse;
  int nb, rs;
  size_t total() const { return plan + tables + o + lse + own_o + own_lse; }
};
size_t pad256(size_t x) { return (x + 255) / 256 * 256; }

TcSizes tc_sizes(int B, int R, int Hkv, int d, int G, int max_group, const Device& di) {
  TcSizes z;
  z.nb = 128 / R < max_group ? 128 / R : max_group;
  z.rs = z.nb * R;
  // A group has at most ceil(rows / tile) row tiles: over all groups B / nb + G.
  const size_t slots = 2 * (((size_t)(B / z.nb) + G) * Hkv + di.sms);
  const size_t own = 2 * ((size_t)B * Hkv + di.sms);
  z.plan = pad256((size_t)B * Hkv * sizeof(int4));
  z.tables = pad256((prefix::tc::Tables::ints(G, B) + 4) * sizeof(int));
  z.o = G ? pad256(slots * z.rs * d * sizeof(float)) : 0;
  z.lse = G ? pad256(slots * z.rs * sizeof(float)) : 0;
  z.own_o = pad256(own * R * d * sizeof(float));
  z.own_lse = pad256(own * R * sizeof(float));
  return z;
}

bool tc_shape(int dtype, int d, int P, int max_pages, int B, int Hq, int Hkv, int G) {
  if (dtype != LLMC_BF16 && dtype != LLMC_F16) return false;
  if (d != 64 && d != 128) return false;
  if (!(P == 8 || P == 16 || P == 32 || P == 64 || P % 128 == 0)) return false;
  const long long R = Hq / Hkv;
  if (R > 128) return false;
  // chunk and slot numbers are 32-bit; a group's row tiles are of at least R rows
  if ((long long)B * Hq >= (1ll << 31)) return false;
  // and so are costs: up to 10 a chunk and 20 a unit, together 15 (chunks + 1) at most
  const long long units = 2ll * B * Hkv + (long long)G * Hkv;
  return units * (((long long)max_pages * P + 127) / 128 + 1) < (1ll << 27);
}
}  // namespace

size_t shared_prefix_workspace_bytes(int B, int Hq, int Hkv, int d, int P, int G, int max_group,
                                     int dtype) {
  const size_t gen = generic_workspace(B, Hq, Hkv, d, G, max_group);
  if (!tc_shape(dtype, d, P, 1, B, Hq, Hkv, G)) return gen;
  const TcSizes z = tc_sizes(B, Hq / Hkv, Hkv, d, G, max_group, device());
  const size_t tc = z.total();
  return tc > gen ? tc : gen;
}

// Launches with programmatic stream serialization: the kernel's start may overlap its
// predecessor, whose results it reads only after griddepcontrol.wait.
template <auto Kern, typename... Args>
static cudaError_t launch_chained(dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                  const Args&... args) {
  if (smem > 48 * 1024) {
    cudaError_t e = allow_shared_memory<Kern>();
    if (e != cudaSuccess) return e;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, Kern, args...);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, int NJ>
static cudaError_t launch_generic_d(prefix::Params p, float* ws, std::string* err,
                                    cudaStream_t stream) {
  namespace gen = prefix::generic;
  const GenericPlan z = generic_plan(p.B, p.Hq, p.Hkv, p.G, p.max_group);
  p.split_g = z.split_g;
  p.split_o = z.split_o;
  int4* groups = reinterpret_cast<int4*>(ws);
  int* seq_s = reinterpret_cast<int*>(groups + p.G);
  p.part_o = ws + generic_tables(p.B, p.G) / sizeof(float);
  p.part_lse = p.part_o + (size_t)(z.split_g + z.split_o) * p.B * p.Hq * p.d;
  const long long blocks = (long long)p.G * z.group_tiles * z.split_g +
                           (long long)p.B * z.seq_tiles * z.split_o;
  if (blocks > INT_MAX || p.Hkv > 65535) {
    *err = "too many row tiles (groups x max_group, sequences) for this shape";
    return cudaErrorInvalidConfiguration;
  }
  cudaError_t e = launch_chained<gen::groups_kernel>(dim3(1), dim3(1024), 0, stream, p, groups,
                                                     seq_s);
  if (e != cudaSuccess) return e;
  e = launch_chained<gen::units_kernel<T, NJ>>(
      dim3((unsigned)blocks, p.Hkv), dim3(gen::kThreads),
      gen::smem_floats(z.rpt, 64 * NJ) * sizeof(float), stream, p, groups, seq_s, z.group_tiles,
      z.seq_tiles, z.rpt);
  if (e != cudaSuccess) return e;
  const long long rows = (long long)p.B * p.Hq;
  return launch_chained<gen::join_kernel<T>>(dim3((unsigned)((rows + 7) / 8)), dim3(256), 0,
                                             stream, p);
}

template <typename T>
static cudaError_t launch_generic(const prefix::Params& p, float* ws, std::string* err,
                                  cudaStream_t stream) {
  if (p.d <= 64) return launch_generic_d<T, 1>(p, ws, err, stream);
  if (p.d <= 128) return launch_generic_d<T, 2>(p, ws, err, stream);
  return launch_generic_d<T, 4>(p, ws, err, stream);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A row-major tensor of 16-bit elements, 64-column boxes with 128-byte swizzle.
static bool encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims,
                   const cuuint64_t* strides, const cuuint32_t* box, int dtype, std::string* err) {
  static EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(ptr);
    return (EncodeTiledFn) nullptr;
  }();
  if (!fn) {
    *err = "cuTensorMapEncodeTiled is not available";
    return false;
  }
  const cuuint32_t estr[3] = {1u, 1u, 1u};
  const CUresult r =
      fn(map, dtype == LLMC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
         (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, estr,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    *err = "cuTensorMapEncodeTiled failed with CUresult " + std::to_string((int)r);
    return false;
  }
  return true;
}

// The pool as rows of d elements; a box is a page or part of one.
static bool encode_pool(CUtensorMap* map, const void* base, long long rows, int d, int box,
                        int dtype, std::string* err) {
  const cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)d * 2};
  const cuuint32_t b[2] = {64u, (cuuint32_t)box};
  return encode(map, base, 2, dims, strides, b, dtype, err);
}

// The same as [half][row][64 columns]: a box is a page of all its halves.
static bool encode_pool_halves(CUtensorMap* map, const void* base, long long rows, int d, int box,
                               int dtype, std::string* err) {
  const cuuint64_t dims[3] = {64u, (cuuint64_t)rows, (cuuint64_t)(d / 64)};
  const cuuint64_t strides[2] = {(cuuint64_t)d * 2, 128u};
  const cuuint32_t b[3] = {64u, (cuuint32_t)box, (cuuint32_t)(d / 64)};
  return encode(map, base, 3, dims, strides, b, dtype, err);
}

// q [B, Hq, d]; a box is the R heads of one KV head of nb sequences, in row order.
static bool encode_q(CUtensorMap* map, const void* base, int B, int Hq, int d, int R, int nb,
                     int dtype, std::string* err) {
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)Hq, (cuuint64_t)B};
  const cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)Hq * d * 2};
  const cuuint32_t b[3] = {64u, (cuuint32_t)R, (cuuint32_t)nb};
  return encode(map, base, 3, dims, strides, b, dtype, err);
}

template <int D, typename T>
static cudaError_t launch_tc(const prefix::Params& p0, void* ws, int dtype, std::string* err,
                             cudaStream_t stream) {
  namespace tc = prefix::tc;
  const Device di = device();
  tc::TcParams tp;
  tp.p = p0;
  prefix::Params& p = tp.p;
  const TcSizes z = tc_sizes(p.B, p.R, p.Hkv, D, p.G, p.max_group, di);
  uint8_t* at = static_cast<uint8_t*>(ws);
  tp.plan = reinterpret_cast<int4*>(at);
  at += z.plan;
  tp.heads = reinterpret_cast<int32_t*>(at);
  tp.tables = tp.heads + 4;
  at += z.tables;
  p.part_o = reinterpret_cast<float*>(at);
  at += z.o;
  p.part_lse = reinterpret_cast<float*>(at);
  at += z.lse;
  tp.own_o = reinterpret_cast<float*>(at);
  at += z.own_o;
  tp.own_lse = reinterpret_cast<float*>(at);
  tp.nb = z.nb;
  tp.rs = z.rs;
  tp.ctas = di.sms;
  CUtensorMap mk, mv, mq, mq1;
  const long long rows = (long long)p.num_pages * p.Hkv * p.P;
  const int box = p.P < tc::kChunk ? p.P : tc::kChunk;
  if (!encode_pool(&mk, p.k_pages, rows, D, box, dtype, err) ||
      !encode_pool_halves(&mv, p.v_pages, rows, D, box, dtype, err) ||
      !encode_q(&mq, p.q, p.B, p.Hq, D, p.R, z.nb, dtype, err) ||
      !encode_q(&mq1, p.q, p.B, p.Hq, D, p.R, 1, dtype, err))
    return cudaErrorInvalidValue;
  // Tables in shared memory, unless the batch is too large for what the tiles leave.
  const size_t fixed = 1024 + tc::Smem<D>::kTables;
  const size_t tables = tc::Tables::ints(p.G, p.B) * sizeof(int);
  cudaError_t e;
  if (fixed + tables > (size_t)di.smem) {
    e = launch_chained<tc::tables_kernel>(dim3(1), dim3(1024), 0, stream, tp);
    if (e != cudaSuccess) return e;
    e = launch_chained<tc::parts_kernel<D, T, true>>(dim3(di.sms), dim3(tc::kThreads), fixed,
                                                     stream, mk, mv, mq, mq1, tp);
  } else {
    e = launch_chained<tc::parts_kernel<D, T, false>>(dim3(di.sms), dim3(tc::kThreads),
                                                      fixed + tables, stream, mk, mv, mq, mq1, tp);
  }
  if (e != cudaSuccess) return e;
  const long long out_rows = (long long)p.B * p.Hq;
  constexpr int per = 256 / (D / 4);
  return launch_chained<tc::join_kernel<D, T>>(dim3((unsigned)((out_rows + per - 1) / per)),
                                               dim3(256), 0, stream, tp);
}

cudaError_t launch_shared_prefix_decode(const void* q, const void* kp, const void* vp,
                                        const int32_t* bt, const int32_t* seq_lens,
                                        const int32_t* starts, const int32_t* shared, void* out,
                                        float* ws, int32_t* status, int B, int Hq, int Hkv, int d,
                                        int P, int max_pages, int num_pages, int G, int max_group,
                                        float scale, int dtype, int flags, std::string* err,
                                        cudaStream_t stream) {
  prefix::Params p;
  p.q = q; p.k_pages = kp; p.v_pages = vp; p.block_table = bt; p.seq_lens = seq_lens;
  p.starts = starts; p.shared = shared; p.out = out; p.status = status;
  p.part_o = nullptr; p.part_lse = nullptr;
  p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.R = Hq / Hkv; p.d = d; p.P = P; p.max_pages = max_pages;
  p.num_pages = num_pages; p.G = G; p.max_group = max_group; p.split_g = p.split_o = 1;
  p.scale_log2 = scale * 1.4426950408889634f;
  auto al = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  if (!(flags & LLMC_DECODE_FORCE_GENERIC) && tc_shape(dtype, d, P, max_pages, B, Hq, Hkv, G) &&
      al(q) && al(kp) && al(vp) && al(out) && scale > 0.f) {
    if (dtype == LLMC_BF16)
      return d == 128 ? launch_tc<128, __nv_bfloat16>(p, ws, dtype, err, stream)
                      : launch_tc<64, __nv_bfloat16>(p, ws, dtype, err, stream);
    return d == 128 ? launch_tc<128, __half>(p, ws, dtype, err, stream)
                    : launch_tc<64, __half>(p, ws, dtype, err, stream);
  }
  if (dtype == LLMC_F32) return launch_generic<float>(p, ws, err, stream);
  if (dtype == LLMC_F16) return launch_generic<__half>(p, ws, err, stream);
  return launch_generic<__nv_bfloat16>(p, ws, err, stream);
}

}  // namespace llmc
