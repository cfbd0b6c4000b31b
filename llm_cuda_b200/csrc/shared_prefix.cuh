// What the shared-prefix kernels have in common: the groups of a batch.
//
// The B sequences of a batch come in G groups of neighbours: group g holds sequences
// [starts[g], starts[g + 1]), and the first shared[g] tokens of its sequences are the same
// tokens.  The shared part that the kernels compute once is
//     s(g) = min(shared[g], the shortest non-empty sequence of the group),
// so no row of it needs a mask, and empty sequences (unused batch rows) cost nothing.  It is
// read through the table row of the group's first non-empty sequence (the leader); what a
// sequence has behind it is read through its own row.  Only the first max_group sequences
// of a group share (the bound that sizes the workspace); later ones, and sequences in no
// group, have s = 0 and read their whole context themselves: same result.
#pragma once

#include "common.cuh"

namespace llmc {
namespace prefix {

struct Params {
  const void* q;               // [B, Hq, d]
  const void* k_pages;         // [num_pages, Hkv, P, d]
  const void* v_pages;
  const int32_t* block_table;  // [B, max_pages]
  const int32_t* seq_lens;     // [B]
  const int32_t* starts;       // [G + 1]
  const int32_t* shared;       // [G]
  void* out;                   // [B, Hq, d]
  float* part_o;
  float* part_lse;
  int32_t* status;
  int B, Hq, Hkv, R, d, P, max_pages, num_pages, G, max_group;   // R = Hq / Hkv
  int split_g, split_o;        // splits of a group's shared tokens, of a sequence's own
  float scale_log2;            // softmax scale * log2(e)
};

// Length of sequence b, within what its table row can address.
__device__ __forceinline__ int seq_len(const Params& p, int b, bool report) {
  const int n = p.seq_lens[b];
  const long long cap = (long long)p.max_pages * p.P;
  if (n < 0 || n > cap) {
    if (report) atomicOr(p.status, kStatusSeqLenRange);
    return n < 0 ? 0 : (int)cap;
  }
  return n;
}

// Whether every group is a range of the batch, by all threads of the block.  If not, nothing is
// shared: the ranges may overlap.
__device__ __forceinline__ bool groups_ok(const Params& p) {
  int bad = 0;
  for (int g = threadIdx.x; g < p.G; g += blockDim.x) {
    const int lo = p.starts[g], hi = p.starts[g + 1];
    bad |= lo < 0 || hi < lo || hi > p.B;
  }
  bad = __syncthreads_or(bad);
  if (bad && threadIdx.x == 0) atomicOr(p.status, kStatusBadGroup);
  return !bad;
}

// Range of group g, clamped to max_group sequences.
__device__ __forceinline__ void group_range(const Params& p, int g, int& lo, int& hi) {
  lo = p.starts[g];
  hi = p.starts[g + 1];
  if (hi - lo > p.max_group) hi = lo + p.max_group;
}

// s(g) and the leader of the group [lo, hi), by all threads of the block.
// `scratch`: two shared ints.
__device__ __forceinline__ void group_prefix(const Params& p, int g, int lo, int hi, int* scratch,
                                             int& s, int& leader) {
  if (threadIdx.x == 0) {
    scratch[0] = 0x7fffffff;
    scratch[1] = 0x7fffffff;
  }
  __syncthreads();
  int mn = 0x7fffffff, first = 0x7fffffff;
  for (int b = lo + (int)threadIdx.x; b < hi; b += blockDim.x) {
    const int n = seq_len(p, b, false);
    if (n > 0) {
      mn = min(mn, n);
      first = min(first, b);
    }
  }
  for (int o = 16; o; o >>= 1) {
    mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
  }
  if ((threadIdx.x & 31) == 0 && first != 0x7fffffff) {
    atomicMin(&scratch[0], mn);
    atomicMin(&scratch[1], first);
  }
  __syncthreads();
  leader = scratch[1] == 0x7fffffff ? -1 : scratch[1];
  s = leader < 0 ? 0 : max(0, min(p.shared[g], scratch[0]));
  __syncthreads();
}

// Group of sequence b (-1: none), by all threads of the block.  `scratch`: a shared int.
__device__ __forceinline__ int group_of(const Params& p, int b, int* scratch) {
  if (threadIdx.x == 0) *scratch = -1;
  __syncthreads();
  for (int g = threadIdx.x; g < p.G; g += blockDim.x) {
    const int lo = p.starts[g], hi = p.starts[g + 1];
    if (b >= lo && b < hi && b - lo < p.max_group) atomicMax(scratch, g);
  }
  __syncthreads();
  const int g = *scratch;
  __syncthreads();
  return g;
}

}  // namespace prefix
}  // namespace llmc
