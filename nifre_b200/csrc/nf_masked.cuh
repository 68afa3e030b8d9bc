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
  const int* units;  // [max_units][12]: key_begin, key_end (virtual), part | n_parts << 16, 0, group fields
  int max_units;
  int unit_tokens;    // the most query tokens of a unit's group
  const int* items;   // [max_items][12]: the tensor-core path's units
  int max_items;
  const int* merge;  // [max_merge][12]: n_parts, first row, kind (1: items), 0, group fields
  int max_merge;
  const int* unit_shares;  // share i: records [i] to [i + 1] - 1
  const int* item_shares;
  const int* counts;  // unit shares, item shares, merge records, units in use
  const uint32_t* masks;
  long long mask_words;
  int tree, window, sinks;
  float scale_log2;
  float* ws;  // partial rows (see part_base): ws_rows x Hq x DP floats
  long long ws_rows;
  int DP;
  int* queue;  // work queue of the persistent kernels; zero between launches
  int* status;
};

struct MaskedGroup {
  int slot, q_row0, ntok, pos0, ctx, n_draft, mask0, part_row0;
};

// Record i of a work list: its own four fields and its group's, in one round trip.
__device__ __forceinline__ int4 load_record(const int* list, int i, MaskedGroup& g) {
  const int4* r = reinterpret_cast<const int4*>(list) + 3 * (long long)i;
  const int4 h = __ldg(r), a = __ldg(r + 1), b = __ldg(r + 2);
  g = MaskedGroup{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  return h;
}

// Units of share i, within the list.
__device__ __forceinline__ int2 load_share(const int* shares, int i, int max_records) {
  return make_int2(max(0, __ldg(shares + i)), min(__ldg(shares + i + 1), max_records));
}

// The group's own bounds against the buffers that the call gave.
__device__ __forceinline__ bool group_ok(const MaskedParams& p, const MaskedGroup& g) {
  if (g.slot < 0 || g.slot >= p.num_slots || g.ntok <= 0 || g.q_row0 < 0 || g.q_row0 > p.rows - g.ntok || g.pos0 < 0)
    return false;
  if (!p.tree) return true;
  const long long words = (long long)((g.n_draft + 31) >> 5);
  return g.n_draft > 0 && g.mask0 >= 0 && g.mask0 + g.ntok * words <= p.mask_words;
}

// And a unit's: its first key, and no more tokens than the launch was sized for.
__device__ __forceinline__ bool unit_ok(const MaskedParams& p, const int4& un, const MaskedGroup& g) {
  return group_ok(p, g) && un.x >= 0 && (un.x & 15) == 0 && g.ntok <= p.unit_tokens;
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
  const int phys = (unsigned)lb < (unsigned)p.max_blocks ? __ldg(btrow + lb) : -1;
  if (phys < 0 || phys >= p.num_blocks) {
    atomicOr(p.status, NF_STATUS_BAD_BLOCK);
    return -1;
  }
  return (long long)phys * p.bs + (k - lb * p.bs);
}

// Partial results of part `part` of a group for one KV head, R = ntok * G rows
// (row = token * G + query head) of DP / 4 float4s: D4 of elements, then (m, l).
// Units store them row by row; items, whose threads hold a row each, store
// float4 c of row r at c * R + r, so that a store is whole lines.  nullptr
// (flagged) where the workspace ends.
__device__ __forceinline__ float* part_base(const MaskedParams& p, const MaskedGroup& g, int part, int kvh) {
  const long long row = (long long)g.part_row0 + (long long)part * g.ntok;
  if (g.part_row0 < 0 || row + g.ntok > p.ws_rows) {
    atomicOr(p.status, NF_STATUS_UNIT_OVERFLOW);
    return nullptr;
  }
  return p.ws + (row * p.Hq + (long long)kvh * g.ntok * p.G) * p.DP;
}

// A softmax state (m, l, values) holds the largest score, the sum of the
// weights 2^(x - m) and the weighted values.  m passes NaN over, so m = -inf
// does not say that nothing was seen: a state whose seen scores are NaN has
// l = NaN, and joins keep it (its weight is 2^-inf = 0, and 0 * NaN is NaN).
// l = 0 is left for no key seen, whose output is 0, and for seen scores that
// are all -inf, whose output is 0 / 0; only then is it asked which.
__device__ __forceinline__ bool sees_any(const MaskedParams& p, const MaskedGroup g, int t) {
  if (!p.tree || g.ctx > 0) return true;  // (a window holds the token itself)
  const int words = (g.n_draft + 31) >> 5;
  uint32_t any = 0;
  for (int i = 0; i < words; ++i) {
    const uint32_t w = __ldg(p.masks + g.mask0 + (long long)t * words + i);
    any |= i + 1 < words || !(g.n_draft & 31) ? w : w & ((1u << (g.n_draft & 31)) - 1);
  }
  return any != 0;
}

// The factor from a final state's weighted values to the output; where l is 0,
// no_output() after the store says whether that 0 / 0 was an output.
__device__ __forceinline__ float state_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ bool no_output(const MaskedParams& p, const MaskedGroup& g, int t, float l) {
  return l == 0.f && sees_any(p, g, t);
}
constexpr float kNaN = __builtin_nanf("");

// The tensor-map path (NF_EUNSUPPORTED, nothing launched: not for this shape).
int launch_masked_tma(const MaskedParams& p, int dtype, void* stream, const char* what);
// The tensor-core items.
int launch_masked_tc(const MaskedParams& p, int dtype, void* stream, const char* what);
// Largest group for a shape, in query rows (0: no such path).
int masked_tma_rows(int dtype, int Hq, int Hkv, int D, int bs);
int masked_tc_rows(int dtype, int Hq, int Hkv, int D, int bs);

}  // namespace nf
