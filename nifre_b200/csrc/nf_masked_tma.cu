// Windowed and tree attention of groups of few query rows (decodes, short
// drafts), for 16-bit pools with head_dim 64 or 128 and a block size that is
// a multiple of 16.  Bound by the key and value bytes.
//
// A CTA owns HG KV heads.  Its producer thread takes (share, head group) tasks
// from a queue and, for the share's units, issues, for each 16-key step of a unit, one tensor copy for
// K and one for V: 16 tokens of one block x HG heads x head_dim, landing
// head-major and 128-byte swizzled.  Steps skip the gap between a window's
// sinks and its last keys, so a group reads its visible keys (rounded to 16)
// and no others.  Consumer warp h computes KV head h for all of the group's
// columns (token x query head) at once: S^T = K Q^T and O^T += V^T P^T with
// mma.sync m16n8k16, the columns as NT tiles of 8, so K and V are read once
// whatever the number of drafted tokens.  (A group has at most 32 query rows;
// tcgen05 with the queries as its rows wants 64 or more, and larger groups go to
// nf_masked_tc.cu.  Keys as the 128 rows and the queries as up to 32 columns
// would fit tcgen05 too; that form has not been built.)
//
// 64 decodes with a window of 4,096 and 64 sinks, 8 KV heads of 128 (1.09 GB):
// 170 us with the merge, the copy bandwidth.  64 with a window of 1,024, 8
// KV heads of 64 (130 MB): 30 us, of which 20 are the bytes and the rest is
// the ramp of 148 CTAs and the merge's launch.  37 trees of 7 tokens (28 columns)
// on 4,096 keys: 72 us with two warps a head of 16 columns each.
//
// Scores, maxima, sums of weights and outputs are float32.  The weights alone
// are rounded, once, to the pools' type for the second product (mma.sync takes
// both operands in one 16-bit type): each is off by half a step at most, 2^-8 of
// it in bf16 and 2^-11 in fp16, and the sum of weights is taken before, so an
// output is off by that much of sum w |v| at most.
//
// Only steps that some column does not wholly see apply the mask.  There the
// weights of unseen keys are 0; as 0 * NaN would still reach the sum, such a
// step looks its value rows over and, where they hold anything not finite,
// adds the seen rows one by one instead.  Scores that are NaN, or all -inf: see
// sees_any.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "nf_internal.h"
#include "nf_masked.cuh"
#include "nf_softmax.cuh"
#include "nf_tma.cuh"

namespace nf {

constexpr int kMtHeader = 1024;
constexpr int kMtMaxStages = 8;

// One 16-key step as the producer describes it to the consumers; the unit's
// fields (from slot on) are set on its first step only.
struct __align__(16) MtStep {
  int u, key0, nv, flags;  // u < 0: no more work; first key, keys before the unit's end, kMt* bits
  int q_row0, ntok, pos0, ctx;
  int n_draft, mask0, part_row0, part;  // part: part | n_parts << 16
  int hg, pad0, pad1, pad2;
};
constexpr int kMtFirst = 1, kMtLast = 2, kMtMasked = 4;

struct MtLaunch {
  int HG, n_hg, stages, stage_bytes, box_bytes, one_box, q_align4;
};

// Byte offset of key row r, 16-byte chunk c, in one head's staged tile.
__device__ __forceinline__ int mt_off(int r, int c) {
  return (c >> 3) * 2048 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// mma.sync and movmatrix as pure functions of their registers (not volatile:
// the scheduler may interleave independent ones with the softmax arithmetic).
template <typename T>
__device__ __forceinline__ void mt_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t mt_transpose(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int D_>
__device__ void mt_producer(const MaskedParams& p, const MtLaunch& L, const CUtensorMap* tk, const CUtensorMap* tv,
                            unsigned char* base) {
  constexpr int NDH = D_ / 64;
  const uint32_t hdr = smem_u32(base);
  auto full = [&](int s) { return hdr + 8 * s; };
  auto empty = [&](int s) { return hdr + 64 + 8 * s; };
  MtStep* recs = reinterpret_cast<MtStep*>(base + 128);
  const uint32_t stage0 = hdr + kMtHeader;
  // the switch to another task needs four dependent round trips (ticket, share,
  // record, block id): each is asked for kGap steps after the one before
  constexpr int kGap = 2, kAhead = 4 * kGap;
  const uint64_t pol = l2_evict_first();  // a share's keys are read by one CTA
  int k = 0, s = 0;
  uint32_t pe = 1;
  bool ok = true;
  // a task: (share, head group); u: the share's unit at work
  int w = blockIdx.x;
  int2 sh = load_share(p.unit_shares, min(w / L.n_hg, p.max_units - 1), p.max_units);
  const int total = min(__ldg(p.counts), p.max_units) * L.n_hg;
  int u = sh.x;
  MaskedGroup g;
  int4 un = load_record(p.units, min(u, p.max_units - 1), g);
  if (w < total && g.slot >= 0 && g.slot < p.num_slots) {  // the block tables are the step's pack's, before that launch
    const int lb = VirtualKeys(p, g).key(un.x) / p.bs;
    if (lb >= 0 && lb < p.max_blocks)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(p.bt + (long long)g.slot * p.max_blocks + lb));
  }
  pdl_wait();
  while (w < total) {
    const int hg = w % L.n_hg, h0 = hg * L.HG;
    const bool more = u + 1 < sh.y;  // the next unit is this share's
    if (u >= sh.y || !unit_ok(p, un, g)) {
      if (u < sh.y) atomicOr(p.status, NF_STATUS_BAD_SLOT);
      if (more) {
        ++u;
      } else {
        w = (int)gridDim.x + atomicAdd(p.queue, 1);
        if (w >= total) break;
        sh = load_share(p.unit_shares, w / L.n_hg, p.max_units);
        u = sh.x;
      }
      un = load_record(p.units, min(u, p.max_units - 1), g);
      continue;
    }
    const VirtualKeys vk(p, g);
    const int v1 = min(un.y, vk.end);
    const int* btrow = p.bt + (long long)g.slot * p.max_blocks;
    const int nsteps = max(1, (v1 - un.x + 15) >> 4);  // (a unit without keys still ends in an epilogue)
    const int ask = nsteps - 1 - min(kAhead, nsteps - 1);
    int wn = more ? w : total, nu_at = u + 1;
    int2 nsh = sh;
    int4 nu = make_int4(0, 0, 0, 0);
    MaskedGroup ng{};
    int have = more ? 2 : 0;  // what is known of the next unit: 1 its task, 2 its place, 3 its record
    for (int i = 0, v = un.x; i < nsteps; ++i, v += 16, ++k) {
      if (i == ask && have == 0) {
        wn = (int)gridDim.x + atomicAdd(p.queue, 1);
        have = 1;
      } else if (i == ask + kGap && have == 1 && wn < total) {
        nsh = load_share(p.unit_shares, wn / L.n_hg, p.max_units);
        nu_at = nsh.x;
        have = 2;
      } else if (have == 2 && (more || i == ask + 2 * kGap)) {
        nu = load_record(p.units, min(nu_at, p.max_units - 1), ng);
        have = 3;
      } else if (have == 3 && i == (more ? 1 : ask + 3 * kGap) && ng.slot >= 0 && ng.slot < p.num_slots) {
        const int lb = VirtualKeys(p, ng).key(nu.x) / p.bs;
        if (lb >= 0 && lb < p.max_blocks)
          asm volatile("prefetch.global.L1 [%0];" ::"l"(p.bt + (long long)ng.slot * p.max_blocks + lb));
      }
      if (!mbar_wait(empty(s), pe, p.status)) {
        ok = false;
        break;
      }
      const int key0 = vk.key(v), key1 = key0 + 15, last_pos = g.pos0 + g.ntok - 1;
      const int lb = key0 / p.bs;
      int phys = (unsigned)lb < (unsigned)p.max_blocks ? __ldg(btrow + lb) : -1;
      // a block that is not there: nothing of it is seen (nv 0 on a masked step), and block 0 stands in
      const bool bad = phys < 0 || phys >= p.num_blocks;
      if (bad) {
        atomicOr(p.status, NF_STATUS_BAD_BLOCK);
        phys = 0;
      }
      const int nv = bad ? 0 : max(0, min(16, v1 - v));
      const bool whole = nv == 16 && (p.tree ? key1 < g.ctx
                                             : key1 <= g.pos0 && (key0 > last_pos - p.window || key1 < p.sinks));
      MtStep& r = recs[s];
      *reinterpret_cast<int4*>(&r) =
          make_int4(u, key0, nv, (i == 0 ? kMtFirst : 0) | (i == nsteps - 1 ? kMtLast : 0) | (whole ? 0 : kMtMasked));
      if (i == 0) {
        reinterpret_cast<int4*>(&r)[1] = make_int4(g.q_row0, g.ntok, g.pos0, g.ctx);
        reinterpret_cast<int4*>(&r)[2] = make_int4(g.n_draft, g.mask0, g.part_row0, un.z);
        r.hg = hg;
      }
      const int off = key0 - lb * p.bs;
      const uint32_t sb = stage0 + s * L.stage_bytes;
      mbar_arrive_expect_tx(full(s), 2 * L.box_bytes);
      if (L.one_box) {
        if constexpr (D_ == 64) {
          tma_load_4d(sb, tk, 0, off, h0, phys, full(s), pol);
          tma_load_4d(sb + L.box_bytes, tv, 0, off, h0, phys, full(s), pol);
        } else {
          tma_load_5d(sb, tk, 0, off, 0, h0, phys, full(s), pol);
          tma_load_5d(sb + L.box_bytes, tv, 0, off, 0, h0, phys, full(s), pol);
        }
      } else {
        for (int h = 0; h < L.HG; ++h)
#pragma unroll
          for (int dh = 0; dh < NDH; ++dh) {
            const uint32_t d = sb + (h * NDH + dh) * 2048;
            if constexpr (D_ == 64) {
              tma_load_4d(d, tk, 0, h0 + h, off, phys, full(s), pol);
              tma_load_4d(d + L.box_bytes, tv, 0, h0 + h, off, phys, full(s), pol);
            } else {
              tma_load_5d(d, tk, 0, dh, h0 + h, off, phys, full(s), pol);
              tma_load_5d(d + L.box_bytes, tv, 0, dh, h0 + h, off, phys, full(s), pol);
            }
          }
      }
      if (++s == L.stages) {
        s = 0;
        pe ^= 1;
      }
    }
    if (!ok) break;
    if (wn < total && have < 3) {  // a short unit
      if (have < 2) {
        nsh = load_share(p.unit_shares, wn / L.n_hg, p.max_units);
        nu_at = nsh.x;
      }
      nu = load_record(p.units, min(nu_at, p.max_units - 1), ng);
    }
    w = wn;
    sh = nsh;
    u = nu_at;
    un = nu;
    g = ng;
  }
  if (ok && mbar_wait(empty(s), pe, p.status)) {
    recs[s].u = -1;
    mbar_arrive(full(s));
    return;
  }
  // a wait ran out: leave no copy in flight into this CTA's shared memory
  for (int j = max(0, k - L.stages); j < k; ++j) mbar_wait(full(j % L.stages), (j / L.stages) & 1, p.status);
}

// A unit as its consumer warp holds it, and the running state of NT tiles of
// 8 columns: column c = 8 j + 2 (lane % 4) (+1) of token c / G.  m is the
// reference the exponents are taken against, 0 while bit 2 j + e of none says
// that the column has seen no key yet.
template <int D_, int NT>
struct MtState {
  static constexpr int KS = D_ / 16;
  uint32_t qf[NT][KS][2];
  float m[NT][2], l[NT][2];
  float o[KS][NT][4];
  uint32_t none;
  uint32_t tok[NT];  // the tokens of columns 8 j + 2 (lane % 4) (low half) and the next (high half)
};

// PT staged 16-key tiles of this warp's head in one update.  With eight
// consumer warps an SM the update's latency and instruction count bound it,
// not its products, so the reference maximum moves only when some score
// exceeds it by more than 8 (one vote a tile pair instead of three shuffles
// a column, and no rescaling of O otherwise: weights stay below 2^8).
template <typename T, int D_, int NT, int PT, bool EARLY>
__device__ __forceinline__ void mt_update(const MaskedParams& p, const MaskedGroup& g, const uint32_t (&kb)[PT],
                                          const uint32_t (&vb)[PT], const int (&key0)[PT], const int (&nv)[PT],
                                          int masked, MtState<D_, NT>& st) {
  constexpr int KS = D_ / 16;
  const int lane = threadIdx.x & 31, tq = lane >> 2, n0 = 2 * (lane & 3);
  // this lane's row and chunk of the fragments; k-step i is an exclusive or of the chunk bits (mt_off(r, 2 i + c))
  const int kr = (lane & 7) + ((lane >> 3) & 1) * 8, vr = (lane & 7) + ((lane >> 4) & 1) * 8;
  const uint32_t ko = mt_off(kr, lane >> 4), vo = mt_off(vr, (lane >> 3) & 1);
  auto step_at = [](uint32_t a, int i) { return (a ^ ((i & 3) << 5)) + (i >> 2) * 2048; };
  float x[PT][NT][4];
  // fragments of both tiles (and of the values) at once where registers allow, else a tile's at a time
  constexpr bool kEarly = EARLY;
  uint32_t kf[kEarly ? PT : 1][KS][4];
#pragma unroll
  for (int t = 0; t < PT; ++t)
#pragma unroll
    for (int j = 0; j < NT; ++j) x[t][j][0] = x[t][j][1] = x[t][j][2] = x[t][j][3] = 0.f;
  if constexpr (kEarly) {
#pragma unroll
    for (int t = 0; t < PT; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        ldsm_x4(step_at(kb[t] + ko, ks), kf[t][ks][0], kf[t][ks][1], kf[t][ks][2], kf[t][ks][3]);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int t = 0; t < PT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j) mt_mma<T>(x[t][j], kf[t][ks], st.qf[j][ks][0], st.qf[j][ks][1]);
  } else {
#pragma unroll
    for (int t = 0; t < PT; ++t) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        ldsm_x4(step_at(kb[t] + ko, ks), kf[0][ks][0], kf[0][ks][1], kf[0][ks][2], kf[0][ks][3]);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < NT; ++j) mt_mma<T>(x[t][j], kf[0][ks], st.qf[j][ks][0], st.qf[j][ks][1]);
    }
  }
  uint32_t vf[kEarly ? PT : 1][KS][4];
  if constexpr (kEarly) {
#pragma unroll
    for (int t = 0; t < PT; ++t)
#pragma unroll
      for (int i = 0; i < KS; ++i)
        ldsm_x4_t(step_at(vb[t] + vo, i), vf[t][i][0], vf[t][i][1], vf[t][i][2], vf[t][i][3]);
  }
  // exponents against the reference; unseen keys -inf
  const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2);
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const uint64_t nm2 = f2_pack(-st.m[j][0], -st.m[j][1]);
#pragma unroll
    for (int t = 0; t < PT; ++t) {
      f2_unpack(f2_fma(f2_pack(x[t][j][0], x[t][j][1]), sc2, nm2), x[t][j][0], x[t][j][1]);
      f2_unpack(f2_fma(f2_pack(x[t][j][2], x[t][j][3]), sc2, nm2), x[t][j][2], x[t][j][3]);
      if (masked >> t & 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = tq + (e >> 1) * 8, tok = e & 1 ? st.tok[j] >> 16 : st.tok[j] & 0xffff;
          if (row >= nv[t] || !sees(p, g, tok, key0[t] + row)) x[t][j][e] = -INFINITY;
        }
      }
      top = fmax3(top, fmaxf(x[t][j][0], x[t][j][1]), fmaxf(x[t][j][2], x[t][j][3]));
    }
  }
  if (__any_sync(0xffffffffu, top > 8.f || st.none)) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(x[0][j][e], x[0][j][2 + e]);
#pragma unroll
        for (int t = 1; t < PT; ++t) mx = fmax3(mx, x[t][j][e], x[t][j][2 + e]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const uint32_t bit = 1u << (2 * j + e);
        const bool first = st.none & bit;  // the first seen keys set the reference, later ones raise it
        const float up = first ? (mx == -INFINITY ? 0.f : mx) : (mx > 8.f ? mx : 0.f);
        const float alpha = first ? 1.f : ex2(-up);
        if (mx != -INFINITY) st.none &= ~bit;
        st.m[j][e] += up;
        st.l[j][e] *= alpha;
#pragma unroll
        for (int t = 0; t < PT; ++t) {
          x[t][j][e] -= up;
          x[t][j][2 + e] -= up;
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          st.o[i][j][e] *= alpha;
          st.o[i][j][2 + e] *= alpha;
        }
      }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < PT; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[t][j][e] = ex2(x[t][j][e]);
      const uint64_t s2 = f2_add(f2_pack(x[t][j][0], x[t][j][1]), f2_pack(x[t][j][2], x[t][j][3]));
      f2_unpack(f2_add(f2_pack(st.l[j][0], st.l[j][1]), s2), st.l[j][0], st.l[j][1]);
    }
#pragma unroll
  for (int t = 0; t < PT; ++t) {
    bool plain = true;
    if (masked >> t & 1) {
      // anything not finite among the value rows? (all exponent bits set, either half of a word)
      constexpr uint32_t EX = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
      bool odd = false;
      for (int c = lane; c < 16 * D_ / 8; c += 32) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(vb[t] + c * 16));
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (w[e] & EX) == EX || ((w[e] >> 16) & EX) == EX;
      }
      plain = !__any_sync(0xffffffffu, odd);
    }
    if (plain) {
      uint32_t pb[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        pb[j][0] = mt_transpose(pack2<T>(x[t][j][0], x[t][j][1]));
        pb[j][1] = mt_transpose(pack2<T>(x[t][j][2], x[t][j][3]));
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        uint32_t(&f)[4] = vf[kEarly ? t : 0][i];
        if constexpr (!kEarly) ldsm_x4_t(step_at(vb[t] + vo, i), f[0], f[1], f[2], f[3]);
#pragma unroll
        for (int j = 0; j < NT; ++j) mt_mma<T>(st.o[i][j], f, pb[j][0], pb[j][1]);
      }
    } else {
      constexpr unsigned kUnseen = 0x80000000u;  // -0: a seen key's weight may have underflowed to 0
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = tq + (e >> 1) * 8, tok = e & 1 ? st.tok[j] >> 16 : st.tok[j] & 0xffff;
          if (row >= nv[t] || !sees(p, g, tok, key0[t] + row)) x[t][j][e] = -0.f;
        }
      for (int row = 0; row < 16; ++row) {
        const int src = (row & 7) * 4 + (lane & 3);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float lo0 = __shfl_sync(0xffffffffu, x[t][j][0], src), lo1 = __shfl_sync(0xffffffffu, x[t][j][1], src);
          const float hi0 = __shfl_sync(0xffffffffu, x[t][j][2], src), hi1 = __shfl_sync(0xffffffffu, x[t][j][3], src);
          const float w0 = row < 8 ? lo0 : hi0, w1 = row < 8 ? lo1 : hi1;
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int d = 16 * i + tq + 8 * h;
              unsigned short b;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(b) : "r"(vb[t] + mt_off(row, d >> 3) + (d & 7) * 2));
              const float v = Elem<T>::to_f(*reinterpret_cast<T*>(&b));
              if (__float_as_uint(w0) != kUnseen) st.o[i][j][2 * h] = fmaf(w0, v, st.o[i][j][2 * h]);
              if (__float_as_uint(w1) != kUnseen) st.o[i][j][2 * h + 1] = fmaf(w1, v, st.o[i][j][2 * h + 1]);
            }
        }
      }
    }
  }
}

template <typename T, int D_, int NT, int CW>
__device__ void mt_consumer(const MaskedParams& p, const MtLaunch& L, unsigned char* base) {
  constexpr int KS = D_ / 16, NDH = D_ / 64;
  // two steps an update (128-wide heads have too few stages to hold two, two warps a head too few registers)
  constexpr bool kPairs = D_ == 64 && CW == 1;
  const int warp = (threadIdx.x >> 5) / CW, c0 = (threadIdx.x >> 5) % CW * (8 * NT);  // KV head, first column
  const int lane = threadIdx.x & 31, tq = lane >> 2, n0 = 2 * (lane & 3);
  const uint32_t hdr = smem_u32(base);
  const MtStep* recs = reinterpret_cast<const MtStep*>(base + 128);
  const uint32_t stage0 = hdr + kMtHeader;
  const int head_region = warp * NDH * 2048;
  MtState<D_, NT> st;
  MaskedGroup g{};
  int part = 0, kvh = 0;
  int s = 0;
  uint32_t ph = 0;
  pdl_wait();  // the queries may come from the launch before this one
  for (;;) {
    if (!mbar_wait(hdr + 8 * s, ph, p.status)) return;
    const int4 r = *reinterpret_cast<const int4*>(recs + s);
    if (r.x < 0) return;
    const int s0 = s;
    if (r.w & kMtFirst) {
      const int4 a = reinterpret_cast<const int4*>(recs + s)[1], b = reinterpret_cast<const int4*>(recs + s)[2];
      g = MaskedGroup{0, a.x, a.y, a.z, a.w, b.x, b.y, b.z};
      part = b.w;
      kvh = recs[s].hg * L.HG + warp;
      const int cols = g.ntok * p.G;
      // the group's queries, straight into the B operand's layout: column 8 j + lane / 4, elements
      // 16 ks + 2 (lane % 4) (+1) and 8 further (once a unit, while the ring fills)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int c = c0 + 8 * j + tq, tok = c / p.G;
        const T* q = reinterpret_cast<const T*>(p.q) + (long long)(g.q_row0 + tok) * p.q_stride +
                     (long long)(kvh * p.G + (c - tok * p.G)) * D_ + n0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v = 0;
            if (c < cols) {
              const T* e = q + 16 * ks + 8 * h;
              if (L.q_align4) {
                v = *reinterpret_cast<const uint32_t*>(e);
              } else {
                v = *reinterpret_cast<const unsigned short*>(e) |
                    (uint32_t)*reinterpret_cast<const unsigned short*>(e + 1) << 16;
              }
            }
            st.qf[j][ks][h] = v;
          }
        st.tok[j] = min((c0 + 8 * j + n0) / p.G, g.ntok - 1) | min((c0 + 8 * j + n0 + 1) / p.G, g.ntok - 1) << 16;
        st.m[j][0] = st.m[j][1] = 0.f;
        st.l[j][0] = st.l[j][1] = 0.f;
      }
      st.none = (1u << (2 * NT)) - 1;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) st.o[i][j][0] = st.o[i][j][1] = st.o[i][j][2] = st.o[i][j][3] = 0.f;
    }
    if (++s == L.stages) {
      s = 0;
      ph ^= 1;
    }
    bool last = r.w & kMtLast;
    const uint32_t sb0 = stage0 + s0 * L.stage_bytes;
    if (kPairs && !last) {
      if (!mbar_wait(hdr + 8 * s, ph, p.status)) return;
      const int4 r1 = *reinterpret_cast<const int4*>(recs + s);
      const int s1 = s;
      const uint32_t sb1 = stage0 + s1 * L.stage_bytes;
      if (++s == L.stages) {
        s = 0;
        ph ^= 1;
      }
      last = r1.w & kMtLast;
      const uint32_t kb[2] = {sb0 + head_region, sb1 + head_region};
      const uint32_t vb[2] = {kb[0] + L.box_bytes, kb[1] + L.box_bytes};
      const int key0[2] = {r.y, r1.y}, nv[2] = {r.z, r1.z};
      mt_update<T, D_, NT, 2, CW == 1>(p, g, kb, vb, key0, nv, (r.w & kMtMasked ? 1 : 0) | (r1.w & kMtMasked ? 2 : 0), st);
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(hdr + 64 + 8 * s0);
        mbar_arrive(hdr + 64 + 8 * s1);
      }
    } else {
      const uint32_t kb[1] = {sb0 + head_region}, vb[1] = {kb[0] + L.box_bytes};
      const int key0[1] = {r.y}, nv[1] = {r.z};
      mt_update<T, D_, NT, 1, false>(p, g, kb, vb, key0, nv, r.w & kMtMasked ? 1 : 0, st);
      __syncwarp();
      if (lane == 0) mbar_arrive(hdr + 64 + 8 * s0);
    }
    if (!last) continue;
    const int cols = g.ntok * p.G, n_parts = part >> 16;
    float* rec = n_parts > 1 ? part_base(p, g, part & 0xffff, kvh) : nullptr;
    uint32_t zero = 0;  // columns whose output is 0 / 0, or nothing
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = st.l[j][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const int c = c0 + 8 * j + n0 + e;
        if (c >= cols) continue;
        const int tok = c / p.G, head = kvh * p.G + (c - tok * p.G);
        if (n_parts == 1) {
          const float inv = state_inverse(l);
          T* dst = reinterpret_cast<T*>(p.out) + (long long)(g.q_row0 + tok) * p.out_stride + (long long)head * D_ + tq;
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            dst[16 * i] = Elem<T>::from_f(st.o[i][j][e] * inv);
            dst[16 * i + 8] = Elem<T>::from_f(st.o[i][j][2 + e] * inv);
          }
          if (l == 0.f) zero |= 1u << (2 * j + e);
        } else if (rec) {
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            const int d = 16 * i + tq;
            __stcg(rec + c * (D_ + 4) + d, st.o[i][j][e]);
            __stcg(rec + c * (D_ + 4) + d + 8, st.o[i][j][2 + e]);
          }
          if (tq == 0)
            __stcg(reinterpret_cast<float2*>(rec + c * (D_ + 4) + D_),
                   make_float2(st.none >> (2 * j + e) & 1u ? -INFINITY : st.m[j][e], l));
        }
      }
    for (; zero; zero &= zero - 1) {
      const int b = __ffs(zero) - 1, c = c0 + 8 * (b >> 1) + n0 + (b & 1), tok = c / p.G;
      if (!no_output(p, g, tok, 0.f)) continue;
      T* dst = reinterpret_cast<T*>(p.out) + (long long)(g.q_row0 + tok) * p.out_stride +
               (long long)(kvh * p.G + (c - tok * p.G)) * D_ + tq;
      for (int i = 0; i < 2 * KS; ++i) dst[8 * i] = Elem<T>::from_f(kNaN);
    }
  }
}

// CW: consumer warps a KV head, each with NT tiles of 8 of the group's columns.
// Measured side by side on 37 trees of 7 tokens over 4096 keys (1B shape, 28
// columns, 310 MB; the build with two warps takes 72 us now): one warp a head
// with all 32 columns 115 us (latency of one update at a time: 10 cycles an
// instruction with two warps a scheduler), the same with 232 registers a thread
// (setmaxnreg) and two steps an update 97 us, two warps a head with 16 columns
// each 82 us (96 registers; more steps an update spill).
template <typename T, int D_, int NT, int CW>
__global__ void __launch_bounds__(32 * ((D_ == 64 ? 8 : 4) * CW + 1), D_ == 64 || CW == 4 ? 1 : 2)
    masked_tma_kernel(const MaskedParams p, const MtLaunch L, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  if (threadIdx.x == 32 * L.HG * CW) {
    tma_prefetch_map(&tk);
    tma_prefetch_map(&tv);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < L.stages; ++s) {
      mbar_init(smem_u32(base) + 8 * s, 1);
      mbar_init(smem_u32(base) + 64 + 8 * s, L.HG * CW);
    }
    fence_mbar_init();
  }
  __syncthreads();
  if (warp < L.HG * CW)
    mt_consumer<T, D_, NT, CW>(p, L, base);
  else if ((threadIdx.x & 31) == 0)
    mt_producer<D_>(p, L, &tk, &tv, base);
  __syncthreads();
  // the last CTA out rewinds the queue (every ticket of every CTA is taken)
  if (threadIdx.x == 0 && atomicAdd(p.queue + 1, 1) == (int)gridDim.x - 1) {
    p.queue[0] = 0;
    p.queue[1] = 0;
    __threadfence();
  }
}

// Query rows of a group: two warps a head hold 16 columns of a 64-wide head
// each, four 8 of a 128-wide one.
int masked_tma_rows(int dtype, int Hq, int Hkv, int D, int bs) {
  if (dtype != NF_BF16 && dtype != NF_F16) return 0;
  if ((D != 64 && D != 128) || bs % 16) return 0;
  const int rows = 32;
  return Hq / Hkv <= rows ? rows : 0;
}

using MtKernel = void (*)(const MaskedParams, const MtLaunch, const CUtensorMap, const CUtensorMap);
template <typename T>
static MtKernel mt_kernel(int D, int cols) {
  if (D == 128)
    return cols <= 8 ? masked_tma_kernel<T, 128, 1, 1> : cols <= 16 ? masked_tma_kernel<T, 128, 1, 2> : masked_tma_kernel<T, 128, 1, 4>;
  return cols <= 8 ? masked_tma_kernel<T, 64, 1, 1> : cols <= 16 ? masked_tma_kernel<T, 64, 2, 1> : masked_tma_kernel<T, 64, 2, 2>;
}

int launch_masked_tma(const MaskedParams& p, int dtype, void* stream, const char* what) {
  if (!masked_tma_rows(dtype, p.Hq, p.Hkv, p.D, p.bs)) return NF_EUNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(p.kp) | reinterpret_cast<uintptr_t>(p.vp)) & 15) return NF_EUNSUPPORTED;
  if (p.unit_tokens * p.G > masked_tma_rows(dtype, p.Hq, p.Hkv, p.D, p.bs)) return NF_EUNSUPPORTED;
  // as many KV heads a CTA as eight warps an SM take; the rest of the SM goes to stages (32 KB each, about
  // 220 KB in flight an SM)
  const int max_hg = p.D == 64 ? 8 : 4;
  int hg = 1;
  for (int h = p.Hkv < max_hg ? p.Hkv : max_hg; h > 1; --h)
    if (p.Hkv % h == 0) {
      hg = h;
      break;
    }
  MtLaunch L;
  L.HG = hg;
  L.n_hg = p.Hkv / hg;
  L.box_bytes = hg * 16 * p.D * 2;
  L.stage_bytes = 2 * L.box_bytes;
  const int cols = p.unit_tokens * p.G;
  const int cw = p.D == 64 ? (cols <= 16 ? 1 : 2) : (cols <= 8 ? 1 : cols <= 16 ? 2 : 4);
  const int want = (p.D == 64 || cw == 4 ? 1 : 2) * (max_hg / hg);
  int stages = (228 * 1024 / want - 1024 - kMtHeader - 1024) / L.stage_bytes;
  L.stages = stages > kMtMaxStages ? kMtMaxStages : stages;
  if (L.stages < 2) return NF_EUNSUPPORTED;
  CUtensorMap tk, tv;
  L.one_box = encode_pool_map(&tk, p.kp, dtype, p.D, p.Hkv, p.bs, p.num_blocks, hg, true) &&
              encode_pool_map(&tv, p.vp, dtype, p.D, p.Hkv, p.bs, p.num_blocks, hg, true);
  if (!L.one_box && !(encode_pool_map(&tk, p.kp, dtype, p.D, p.Hkv, p.bs, p.num_blocks, hg, false) &&
                      encode_pool_map(&tv, p.vp, dtype, p.D, p.Hkv, p.bs, p.num_blocks, hg, false)))
    return NF_EUNSUPPORTED;
  L.q_align4 = (reinterpret_cast<uintptr_t>(p.q) % 4 == 0) && p.q_stride % 2 == 0;
  const MtKernel kern = dtype == NF_BF16 ? mt_kernel<__nv_bfloat16>(p.D, cols) : mt_kernel<__half>(p.D, cols);
  const int threads = (hg * cw + 1) * 32, smem = kMtHeader + L.stages * L.stage_bytes + 1024;
  int per_sm = 1;
  cudaError_t e = prepare_launch(reinterpret_cast<const void*>(kern), smem, threads, &per_sm);
  if (e != cudaSuccess) return fail(NF_ECUDA, "%s: smem attribute: %s", what, cudaGetErrorString(e));
  long long grid = (long long)sm_count() * per_sm;
  const long long need = (long long)p.max_units * L.n_hg;
  if (need < grid) grid = need;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, p, L, tk, tv);
  if (e != cudaSuccess) return fail(NF_ECUDA, "%s: launch: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace nf
