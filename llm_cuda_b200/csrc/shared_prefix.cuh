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

}  // namespace prefix
}  // namespace llmc
