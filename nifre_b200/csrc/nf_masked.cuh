// Attention of a step's queries over part of their sequence's cached keys:
// the last `window` keys and the first `sinks` keys (window), or the cached
// context and the drafted tokens a bit mask names (tree).  Records and
// device helpers shared by the kernels of nf_masked*.cu.
//
// Query token i of a sequence stands at position p.  It sees key k when
//   window:  k <= p  and  (k > p - window  or  k < sinks)
//   tree:    k < ctx  or  bit k - ctx of the token's mask row is set
// and its output is sum_k softmax_k(q . k * scale) v_k over the keys it sees
// (0 when it sees none).  Keys a token does not see contribute nothing,
// whatever their rows hold (NaN and infinities included).
//
// A group is a run of consecutive query tokens of one sequence; its keys are
// numbered without the gap between the sinks and the window ("virtual" keys,
// a whole number of 16-key blocks left out), and cut into units: parts of the
// group's keys, merged afterwards where there are several (split-K).
#pragma once

#include <math.h>

#include "nf_common.cuh"

namespace nf {

struct MaskedParams {
  char* out;
  long long out_stride;
  const char* q;
  long long q_stride;
  const char* kp;
  const char* vp;
  int rows;  // rows of q and out
  int Hq, Hkv, D, G, bs, num_blocks;
  const int* bt;
  int num_slots, max_blocks;
  const int* groups;  // [max_groups][8]: slot, q_row0, ntok, pos0, ctx, n_draft, mask0, part_row0
  int max_groups;
  const int* units;  // [max_units][4]: group, key_begin, key_end (virtual), part | n_parts << 16
  int max_units;
  int unit_tokens;    // the most query tokens of a unit's group
  const int* items;   // [max_items][4]: the tensor-core path's units
  int max_items;
  const int* merge;  // [max_merge][4]: q_row, part_row0, n_parts, rows between an item's parts
  int max_merge;
  const int* counts;  // units, tensor-core items, merge rows, partial rows
  const uint32_t* masks;
  long long mask_words;
  int tree, window, sinks;
  float scale_log2;
  float* ws;  // partial rows [part row][Hq][DP]: acc[D], m, l
  long long ws_rows;
  int DP;
  int* queue;  // work queue of the persistent kernels; zero between launches
  int* status;
};

struct MaskedGroup {
  int slot, q_row0, ntok, pos0, ctx, n_draft, mask0, part_row0;
};

__device__ __forceinline__ MaskedGroup load_group(const MaskedParams& p, int g) {
  const int4* r = reinterpret_cast<const int4*>(p.groups) + 2 * g;
  const int4 a = __ldg(r), b = __ldg(r + 1);
  return MaskedGroup{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

// The group's own bounds against the buffers that the call gave.
__device__ __forceinline__ bool group_ok(const MaskedParams& p, const MaskedGroup& g) {
  if (g.slot < 0 || g.slot >= p.num_slots || g.ntok <= 0 || g.q_row0 < 0 || g.q_row0 > p.rows - g.ntok || g.pos0 < 0)
    return false;
  if (!p.tree) return true;
  const long long words = (long long)((g.n_draft + 31) >> 5);
  return g.n_draft > 0 && g.mask0 >= 0 && g.mask0 + g.ntok * words <= p.mask_words;
}

// Virtual keys of a group: 16-key blocks wholly before the first token's
// window and past the sinks are left out.  Virtual key v is key v for
// v < kept, else v + gap; `end` virtual keys in all.
struct VirtualKeys {
  int kept, gap, end;
  __device__ __forceinline__ VirtualKeys(const MaskedParams& p, const MaskedGroup& g) {
    if (p.tree) {
      kept = gap = 0;
      end = g.ctx + g.n_draft;
    } else {
      const int lo = max(0, g.pos0 - p.window + 1) & ~15;
      kept = min((p.sinks + 15) & ~15, lo);
      gap = lo - kept;
      end = g.pos0 + g.ntok - gap;
    }
  }
  __device__ __forceinline__ int key(int v) const { return v < kept ? v : v + gap; }
};

// Whether token t of group g sees key k.
__device__ __forceinline__ bool sees(const MaskedParams& p, const MaskedGroup& g, int t, int k) {
  if (p.tree) {
    if (k < g.ctx) return true;
    const int j = k - g.ctx;
    if (j >= g.n_draft) return false;
    const int words = (g.n_draft + 31) >> 5;
    return (__ldg(p.masks + g.mask0 + t * words + (j >> 5)) >> (j & 31)) & 1u;
  }
  const int pos = g.pos0 + t;
  return k <= pos && (k > pos - p.window || k < p.sinks);
}

// Pool row of key k of a slot (-1: no such block; flagged).
__device__ __forceinline__ long long key_row(const MaskedParams& p, const int* btrow, int k) {
  const int lb = k / p.bs;
  const int phys = lb < p.max_blocks ? __ldg(btrow + lb) : -1;
  if (phys < 0 || phys >= p.num_blocks) {
    atomicOr(p.status, NF_STATUS_BAD_BLOCK);
    return -1;
  }
  return (long long)phys * p.bs + (k - lb * p.bs);
}

// Partial record of (partial row, query head).
__device__ __forceinline__ float* part_record(const MaskedParams& p, long long row, int head) {
  return p.ws + (row * p.Hq + head) * p.DP;
}

// The tensor-map path (NF_EUNSUPPORTED, nothing launched: not for this shape).
int launch_masked_tma(const MaskedParams& p, int dtype, void* stream, const char* what);
// The tensor-core items.
int launch_masked_tc(const MaskedParams& p, int dtype, void* stream, const char* what);
// Largest group for a shape, in query rows (0: no such path).
int masked_tma_rows(int dtype, int Hq, int Hkv, int D, int bs);
int masked_tc_rows(int dtype, int Hq, int Hkv, int D, int bs);

}  // namespace nf
