// wr_attention.cuh — what the attention kernels share: their arguments, the
// split of the work over warps, and the layout of the partial results.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "wr_common.cuh"
#include "wr_internal.h"

namespace wr {

constexpr int kUnitTokens = 16;  // keys that a warp takes at a time

// The rows of a segment (one sequence, or the shared prefix with the tokens
// of all sequences) are its (token, query head of the key head's group)
// pairs, in tiles of MR rows; its keys are cut into units of kUnitTokens.
// All units of a launch, in the order (sequence, key head, row tile, unit),
// are dealt to the warps in ranges of equal length, whatever the lengths of
// the sequences are: a range that covers a (row tile)'s keys whole leaves its
// result in `home`, one that starts at the tile's first unit and stops short
// in the warp's slot 1, one that starts further on in its slot 0.  Which
// warps hold a tile's pieces follows from the ranges alone.
struct AttnSplit {
  int64_t units;   // of the launch
  int64_t ranges;  // warps with a range: min(warps, units)
};
// Quotients of 32 bits where they do (a 64-bit division is some hundred
// instructions).
__host__ __device__ inline int64_t quotient(int64_t a, int64_t b) {
  return ((uint64_t)a | (uint64_t)b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
__host__ __device__ inline int64_t range_start(const AttnSplit& s, int64_t w) {
  return quotient(w * s.units, s.ranges);
}
// The warp whose range holds unit u.
__host__ __device__ inline int64_t range_of(const AttnSplit& s, int64_t u) {
  return quotient((u + 1) * s.ranges - 1, s.units);
}

// Partial results: unnormalised sums O [dim] in fp32 with (m, l): m the
// maximum of the scores in units of log2, l the sum of 2^(score - m).
struct AttnPartials {
  float* piece;      // [warps][2][MR][dim]
  float2* piece_ml;  // [warps][2][MR]
};

struct AttnArgs {
  const void* q;
  const void *kc, *vc;
  int64_t q_ts, q_hs, page_stride, head_stride, slot_stride;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* q_start;
  const int32_t* prefix_pages;
  int num_pages, page_size, page_shift;  // page_shift < 0: not a power of two
  int T, B, hq, hkv, group, dim, table_width;
  int prefix;        // keys of the shared prefix that each sequence reads with its own
  int lead;          // > 0: segment 0 is the prefix of that many keys with all T tokens'
                     // rows, and the sequences come behind it
  int direct;        // nothing else adds to the sequences' rows: whole tiles are final
  float scale_log2;
  AttnPartials part;
  float* home;       // [T * hq][dim]
  float2* home_ml;   // [T * hq]
  float* lead_home;  // the same of segment 0
  float2* lead_home_ml;
  int64_t* seg_unit; // [segments + 1] first unit of each segment, and all of them
  int32_t* token_seq;  // [T] sequence of each token, -1: none
  int4* ends;        // null, or [warps] the tile that a warp begins and leaves to the next: segment,
                     // key head, row tile and its last unit there (-1: it leaves none)
  void* out;
  float* lse;
};

// The prefix on the tensor cores (wr_attn_prefix.cu): units of 128 keys, row
// tiles of 128 or 256 rows, one CTA a range.
constexpr int kPrefixUnit = 128;
bool prefix_tiles_ok(const AttnProblem& p);
wr_status_t launch_attn_prefix(const AttnProblem& p, const AttnArgs& a, int row_tile, int grid,
                               cudaStream_t stream);

// Keys that a page holds: index and rest.
WR_DEVINL void split_page(int j, int page_size, int shift, int& page, int& row) {
  page = shift >= 0 ? j >> shift : j / page_size;
  row = j - (shift >= 0 ? page << shift : page * page_size);
}

struct Segment {
  int q0, nq;  // first token, tokens asked
  int len;     // own keys in the cache
  int prefix;  // keys of the prefix before them
};
__host__ __device__ inline int segments(const AttnArgs& a) { return a.B + (a.lead > 0); }
// q_start and lens come from device memory: whatever they hold, the values
// used lie inside q and the table.
WR_DEVINL Segment segment(const AttnArgs& a, int i) {
  Segment s;
  if (a.lead > 0 && i-- == 0) {
    s.q0 = 0; s.nq = a.T; s.len = 0; s.prefix = a.lead;
    return s;
  }
  if (a.q_start) {
    const int lo = min(max(__ldg(a.q_start + i), 0), a.T);
    const int hi = min(max(__ldg(a.q_start + i + 1), lo), a.T);
    s.q0 = lo; s.nq = hi - lo;
  } else {
    s.q0 = i; s.nq = 1;
  }
  s.len = (int)min((int64_t)max(__ldg(a.lens + i), 0), (int64_t)a.table_width * a.page_size);
  s.prefix = a.prefix;
  return s;
}
template <int MR>
WR_DEVINL int row_tiles(const AttnArgs& a, const Segment& s) { return (s.nq * a.group + MR - 1) / MR; }
// A segment without keys still has one unit, so that its rows are written.
WR_DEVINL int key_units(const Segment& s) { return max(1, (s.prefix + s.len + kUnitTokens - 1) / kUnitTokens); }

}  // namespace wr
