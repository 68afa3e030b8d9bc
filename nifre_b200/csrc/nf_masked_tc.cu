// Windowed and tree attention of larger groups (prefill chunks, wide drafts)
// on fifth-generation tensor cores (tcgen05, tensor memory), for 16-bit pools
// with head_dim 64 or 128 and a block size that is a multiple of 16.
//
// An item is (unit, KV head), a task (share of units, KV head).  Up to 256 query rows (row = token * G + query
// head), as two 128-row halves, against the unit's part of the group's
// virtual keys in tiles of 128.  Each 16-key block of a tile has its own
// place in the pools, so the gap between a window's sinks and its last keys
// costs nothing: tiles hold visible keys (rounded to 16) only.
//
//   producer warp: tensor copies of the queries and of K and V tiles (a
//     block's 16 tokens a copy, two for the K of 128-wide heads) into rings;
//   MMA warp: S_h = Q_h K^T (M = N = 128) into tensor memory, then
//     O_h += P_h V with P_h from tensor memory;
//   two softmax warpgroups (thread = row), one per half;
//   two value warps: the value rows of tiles under the mask (below).
//
// An item of one half and several tiles (a draft of up to 128 rows) would
// leave the second warpgroup idle and be bound by the first one's
// exponentials; there both halves take the same queries, half h the tiles
// j = h (mod 2) with an accumulator of its own, joined at the item's end.
//
// The mask is applied only on tiles that some row does not wholly see: each
// row's 128 truth values are built as four words (two runs for a window, the
// shifted mask words for a tree).  Unseen keys get weight 0; as 0 * NaN would
// still reach the sum, the value warps look over a masked tile's value rows
// before P V reads them: rows that are not finite are zeroed, and where some row of the
// item does see one of them, the item's rows are computed again one by one
// (slow, and right: such values are rare and wrong already).  So they are where
// a block of the item is not there.  Scores that are NaN, or all -inf: see sees_any.
//
// Scores, maxima, sums of weights, accumulators and partial results are float32.
// The weights alone are rounded, once, to the pools' type for P V (both
// operands have one 16-bit type): each is off by half a step at most, 2^-8 of it
// in bf16 and 2^-11 in fp16, and the sum of weights is taken before.
//
// What is known of its bounds, from copies of the kernel that leave work out.
// Heads of 64 (4 chunks of 512 tokens, windows of 1,024, 32 heads): 46 us, 37
// without the exponentials, which are thus 9 of them.  A pair of tiles takes
// 3,100 cycles (2,048 on the special-function unit, 1,024 in products), about 29
// us for the two items of nine pairs an SM has; the rest is outside that loop:
// the start and the epilogue of the items, which nothing hides, edge tiles
// under the mask, and the second turn of 256 items on 148 SMs.  Heads
// of 128 (a chunk of 2,048 tokens, window 4,096, 32 heads): 160 us in calls one
// after another (860 TFLOP/s), 140 in replays short enough for the clock to
// stay up; first the copies of 16-key blocks (139 -> 128 us with an eighth of
// them; 144 before a value block was one copy instead of two), then the chain S,
// weights, P V of a half.  Parts to even the two turns out cost as much in merging.
// 16 trees of 32 tokens on contexts up to 4,096, 32 heads of 64: 44 us, where the
// copies and the transitions between items weigh most.  Taken and dropped: two
// threads a row (the exchange of their maxima costs 450 cycles a tile), the next
// scores loaded before the weights are stored, S in two products of 64 keys.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "nf_internal.h"
#include "nf_masked.cuh"
#include "nf_softmax.cuh"
#include "nf_tma.cuh"
#include "nf_umma.cuh"

namespace nf {

template <int D_>
struct TcCfg {
  static constexpr uint32_t TILE = 128 * D_ * 2;  // a 128-row Q half, or a 128-key K or V tile
  static constexpr int QST = D_ == 64 ? 2 : 1;    // Q ring (an item's halves per stage)
  static constexpr int KST = D_ == 64 ? 4 : 2;
  static constexpr int VST = D_ == 64 ? 5 : 3;    // (held one tile longer than K)
  static constexpr int V_BLOCK = 16 * D_ * 2;     // 16 keys of a V tile: 128-byte rows, [d / 64][key]
  static constexpr bool P_ALIAS = D_ == 128;      // P_h over the first 64 columns of S_h (no room left)
  static constexpr uint32_t Q_OFF = 2048;         // after the header
  static constexpr uint32_t K_OFF = Q_OFF + QST * 2 * TILE;
  static constexpr uint32_t V_OFF = K_OFF + KST * TILE;
  static constexpr uint32_t SMEM = 1024 + V_OFF + VST * TILE;  // + alignment slack
  static constexpr int THREADS = 384;  // warp 0 producer, 1 MMA, 2-3 values, 4-7 half 0, 8-11 half 1
  // setmaxnreg split of the launch's 384 x 168 registers
  static constexpr int REGS_CTRL = 72, REGS_SOFTMAX = 216;
  static_assert(REGS_CTRL * 128 + REGS_SOFTMAX * 256 <= 168 * THREADS, "register split exceeds the launch");
  static constexpr uint32_t TMEM_COLS = 512;
  static __device__ __forceinline__ uint32_t s_col(int h) { return h * 128; }
  static __device__ __forceinline__ uint32_t o_col(int h) { return 256 + h * D_; }
  static __device__ __forceinline__ uint32_t p_col(int h) { return P_ALIAS ? h * 128 : 2 * (128 + D_) + h * 64; }
};

constexpr int kTcItemRing = 4;
constexpr uint32_t kTcTmemPtr = 512, kTcPoison = 528, kTcSlots = 576, kTcStats = 1024;

struct TcBars {
  uint32_t hdr;
  __device__ explicit TcBars(uint32_t h) : hdr(h) {}
  __device__ uint32_t k_full(int s) const { return hdr + 8 * s; }
  __device__ uint32_t k_empty(int s) const { return hdr + 64 + 8 * s; }
  __device__ uint32_t v_full(int s) const { return hdr + 128 + 8 * s; }
  __device__ uint32_t v_empty(int s) const { return hdr + 192 + 8 * s; }
  __device__ uint32_t s_full(int h) const { return hdr + 256 + 8 * h; }
  __device__ uint32_t s_free(int h) const { return hdr + 272 + 8 * h; }
  __device__ uint32_t p_full(int h) const { return hdr + 288 + 8 * h; }
  __device__ uint32_t o_done(int h) const { return hdr + 304 + 8 * h; }
  __device__ uint32_t q_full(int s) const { return hdr + 320 + 8 * s; }
  __device__ uint32_t q_empty(int s) const { return hdr + 336 + 8 * s; }
  __device__ uint32_t item_full(int s) const { return hdr + 384 + 8 * s; }
  __device__ uint32_t item_empty(int s) const { return hdr + 416 + 8 * s; }
  __device__ uint32_t v_clean(int s) const { return hdr + 464 + 8 * s; }  // (to 504) a masked tile's values are looked over
  __device__ uint32_t join_full() const { return hdr + 448; }   // half 1's accumulator and statistics are in place
  __device__ uint32_t join_empty() const { return hdr + 456; }  // half 0 has read them
};

// One work item as every role sees it: the producer derives it once, the
// others read the fields they need from its slot in shared memory.
struct __align__(16) TcItem {
  int kvh, k0, k1, part;  // KV head (-1: no more items), virtual keys [k0, k1), part | n_parts << 16
  int nkt, n_half;
  int whole0, whole1;  // tiles that every row sees wholly: [whole0, whole1)
  MaskedGroup g;
  int kept, gap, dup, bad;  // (kept, gap: VirtualKeys)
  TcItem() = default;
  __device__ TcItem(const MaskedParams& p, int head, int4 un, const MaskedGroup& gr, int TT) : g(gr) {
    const VirtualKeys vk(p, gr);
    kvh = head;
    k0 = un.x;
    k1 = min(un.y, vk.end);
    part = un.z;
    kept = vk.kept;
    gap = vk.gap;
    bad = head < 0 || !group_ok(p, g) || k0 < 0 || (k0 & 15) || k0 >= k1 || g.ntok > 2 * TT;
    nkt = bad ? 0 : (k1 - k0 + 127) >> 7;
    n_half = g.ntok > TT ? 2 : 1;
    dup = n_half == 1 && nkt > 1;
    const int v_lo = p.tree ? 0 : max(kept, g.pos0 + g.ntok - p.window - gap);
    const int v_hi = min(k1, p.tree ? g.ctx : g.pos0 + 1 - gap);
    whole0 = max(v_lo - k0 + 127, 0) >> 7;
    whole1 = max(v_hi - k0, 0) >> 7;
  }
  __device__ __forceinline__ int key(int v) const { return v < kept ? v : v + gap; }
  __device__ __forceinline__ bool active(int h, int j) const {
    return j >= 0 && j < nkt && (dup ? (j & 1) == h : h < n_half);
  }
  // tiles of half h
  __device__ __forceinline__ int tiles(int h) const {
    return dup ? (nkt + 1 - h) >> 1 : (h < n_half ? nkt : 0);
  }
  // whether some row of the group may not see the whole of tile j
  __device__ __forceinline__ bool masked(int j) const { return j < whole0 || j >= whole1; }
};
static_assert(sizeof(TcItem) == 80 && kTcSlots + kTcItemRing * sizeof(TcItem) <= kTcStats, "item slots");

// Bits [lo, hi) of word w of a 128-bit row.
__device__ __forceinline__ uint32_t run_bits(int lo, int hi, int w) {
  lo = max(lo - 32 * w, 0);
  hi = min(hi - 32 * w, 32);
  if (hi <= lo) return 0u;
  return (0xffffffffu >> (32 - hi)) & (0xffffffffu << lo);
}

// Truth values of token t's row over tile j: bit i of word i / 32 for key i.
__device__ __forceinline__ void row_bits(const MaskedParams& p, const TcItem& w, int t, int j, uint32_t (&bits)[4]) {
  const int v0 = w.k0 + 128 * j, lim = w.k1 - v0;
  if (p.tree) {
    const int words = (w.g.n_draft + 31) >> 5;
    const uint32_t* row = p.masks + w.g.mask0 + (long long)t * words;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int s = v0 + 32 * q - w.g.ctx;  // drafted token of the word's first bit
      uint32_t b;
      if (s <= -32) {
        b = 0xffffffffu;
      } else if (s < 0) {
        b = (0xffffffffu >> (32 + s)) | (__ldg(row) << -s);
      } else {
        const int i = s >> 5, sh = s & 31;
        const uint32_t a = i < words ? __ldg(row + i) : 0u, c = i + 1 < words ? __ldg(row + i + 1) : 0u;
        b = __funnelshift_r(a, c, sh);
      }
      bits[q] = b & run_bits(0, lim, q);
    }
    return;
  }
  const int pos = w.g.pos0 + t;
  const int a = (w.gap ? p.sinks : min(p.sinks, pos + 1)) - v0;
  const int b = max(pos - p.window + 1, 0) - w.gap - v0, c = min(pos - w.gap - v0 + 1, lim);
#pragma unroll
  for (int q = 0; q < 4; ++q) bits[q] = run_bits(0, min(a, lim), q) | run_bits(max(b, 0), c, q);
}

// Whether any token of the group sees the key.
__device__ __noinline__ bool seen_by_any(const MaskedParams& p, const MaskedGroup g, int key) {
  for (int t = 0; t < g.ntok; ++t)
    if (sees(p, g, t, key)) return true;
  return false;
}

// The ring that hands items to the CTA's warps.
struct TcRing {
  const TcBars& bar;
  TcItem* slots;
  Ring r;
  __device__ TcRing(const TcBars& b, unsigned char* base) : bar(b), slots(reinterpret_cast<TcItem*>(base + kTcSlots)) {}
  // the item in slot st (until release)
  __device__ const TcItem& item(int st) const { return slots[st]; }
  // waits for the next item: its slot (-1 at the end, or when the wait ran out)
  __device__ int next(int* status) {
    if (!mbar_wait(bar.item_full(r.st), r.ph, status)) return -1;
    return slots[r.st].kvh < 0 ? -1 : r.st;
  }
  __device__ void release() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar.item_empty(r.st));
    r.next(kTcItemRing);
  }
};

// The producer's side: the next unit of the (share, KV head) task at work, or
// the next task's first.
struct TcClaim {
  int task = -1, u = 0;
  int2 sh = make_int2(0, 0);
};
__device__ __forceinline__ bool tc_claim(const MaskedParams& p, TcRing& ring, int tasks, TcClaim& cl, int TT,
                                         TcItem& w) {
  const int lane = threadIdx.x & 31;
  while (++cl.u >= cl.sh.y && cl.task < tasks) {
    int pos = blockIdx.x;  // the first task is the CTA's own, the queue hands out the rest
    if (cl.task >= 0) {
      if (lane == 0) pos = (int)gridDim.x + atomicAdd(p.queue + 2, 1);
      pos = __shfl_sync(0xffffffffu, pos, 0);
    }
    cl.task = pos;
    if (pos >= tasks) break;
    cl.sh = load_share(p.item_shares, pos / p.Hkv, p.max_items);
    cl.u = cl.sh.x - 1;
  }
  const int head = cl.task < tasks ? cl.task % p.Hkv : -1;
  int4 un = make_int4(0, 0, 0, 0);
  MaskedGroup g{};
  if (head >= 0) un = load_record(p.items, cl.u, g);
  w = TcItem(p, head, un, g, TT);
  if (!mbar_wait(ring.bar.item_empty(ring.r.st), ring.r.ph ^ 1, p.status)) return false;
  if (lane == 0) {
    ring.slots[ring.r.st] = w;
    mbar_arrive(ring.bar.item_full(ring.r.st));
  }
  __syncwarp();
  ring.r.next(kTcItemRing);
  return head >= 0;
}

// Block id of 16-key block `lane` (< 8) of tile j and its first key; -1: none there.
__device__ __forceinline__ int tc_block(const MaskedParams& p, const TcItem& w, const int* btrow, int j, int lane,
                                        int& key) {
  const int v = w.k0 + (j * 8 + lane) * 16;
  key = w.key(v);
  const int lb = key / p.bs;
  if (lane >= 8 || v >= w.k1) return 0;
  return (unsigned)lb < (unsigned)p.max_blocks ? __ldg(btrow + lb) : -1;
}

// Copies of one 128-key K or V tile, lane b < nb the 16-key block b.  A block
// of a 128-wide head is two boxes of 64 elements a K tile, whose rows are
// evenly spaced for S, and one box of both a V tile, where a block is one k-step
// of P V (fewer copies: 2 KB a copy is what the copies' rate suffers from).
template <int D_, bool V>
__device__ __forceinline__ void tc_load(const MaskedParams& p, const CUtensorMap* tm, uint32_t dst0, uint32_t full,
                                        int phys, int key, int nb, int kvh, uint64_t pol, int lane,
                                        volatile int* poison, int seq) {
  constexpr int NDH = D_ / 64;
  if (lane == 0) mbar_arrive_expect_tx(full, nb * NDH * 2048);
  __syncwarp();
  if (lane < nb) {
    const int off = key % p.bs;
    if (phys < 0 || phys >= p.num_blocks) {
      atomicOr(p.status, NF_STATUS_BAD_BLOCK);
      phys = 0;  // stands in: the item's rows are computed again without the block
      poison[seq & 7] = seq;
    }
    if constexpr (D_ == 64) {
      tma_load_4d(dst0 + lane * 2048, tm, 0, kvh, off, phys, full, pol);
    } else if constexpr (V) {
      tma_load_5d(dst0 + lane * 4096, tm, 0, off, 0, kvh, phys, full, pol);
    } else {
#pragma unroll
      for (int dh = 0; dh < NDH; ++dh)
        tma_load_5d(dst0 + dh * 128 * 128 + lane * 2048, tm, 0, dh, kvh, off, phys, full, pol);
    }
  }
}

// Queries whose rows no tensor copy takes (not 16-byte aligned): element
// loads into the copies' swizzled layout.
template <typename T, int D_>
__device__ void tc_load_queries(const MaskedParams& p, const TcItem& w, int TT, uint32_t dst0, uint32_t full, int lane) {
  constexpr int NDH = D_ / 64;
  const int rows = w.n_half * TT * p.G, half = TT * p.G;
  for (int c = lane; c < rows * NDH * 8; c += 32) {
    const int R = c / (NDH * 8), rest = c % (NDH * 8), h = R / half, row = R - h * half;
    const int tok = h * TT + row / p.G, hd = row % p.G;
    uint32_t v[4] = {0, 0, 0, 0};
    if (tok < w.g.ntok) {
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p.q) + (long long)(w.g.q_row0 + tok) * p.q_stride +
                                (long long)(w.kvh * p.G + hd) * D_ + rest * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
    }
    const uint32_t dst = dst0 + h * TcCfg<D_>::TILE + (rest >> 3) * 128 * 128 + row * 128 + (((rest & 7) ^ (row & 7)) << 4);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                 : "memory");
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) mbar_arrive(full);
}

template <typename T, int D_>
__device__ void tc_producer(const MaskedParams& p, int TT, bool q_tma, const CUtensorMap* tq, const CUtensorMap* tk,
                            const CUtensorMap* tv, const TcBars& bar, unsigned char* base, uint32_t q_s, uint32_t k_s,
                            uint32_t v_s, int tasks, TcRing& ring) {
  using C = TcCfg<D_>;
  constexpr int NDH = D_ / 64;
  const int lane = threadIdx.x & 31;
  const uint64_t pol = l2_evict_last(), pol_q = l2_evict_first();
  volatile int* poison = reinterpret_cast<volatile int*>(base + kTcPoison);
  int seq = 0;
  Ring qr, kr, vr;
  TcClaim claim;
  TcItem w;
  pdl_wait();  // queries, keys and values may come from the launch before this one
  while (tc_claim(p, ring, tasks, claim, TT, w)) {
    if (w.bad) {
      if (lane == 0) atomicOr(p.status, NF_STATUS_BAD_SLOT);
      continue;
    }
    ++seq;
    const int* btrow = p.bt + (long long)w.g.slot * p.max_blocks;
    int key, cur = tc_block(p, w, btrow, 0, lane, key);
    if (!mbar_wait(bar.q_empty(qr.st), qr.ph ^ 1, p.status)) return;
    const uint32_t q_full = bar.q_full(qr.st), q_dst = q_s + qr.st * 2 * C::TILE;
    if (q_tma) {
      const int nq = w.n_half * NDH;
      if (lane == 0) mbar_arrive_expect_tx(q_full, nq * TT * p.G * 128);
      __syncwarp();
      if (lane < nq) {
        const int h = lane / NDH, dh = lane - h * NDH;
        const uint32_t dst = q_dst + h * C::TILE + dh * 128 * 128;
        const int row0 = w.g.q_row0 + h * TT;
        if constexpr (D_ == 64)
          tma_load_3d(dst, tq, 0, w.kvh * p.G, row0, q_full, pol_q);
        else
          tma_load_4d(dst, tq, 0, dh, w.kvh * p.G, row0, q_full, pol_q);
      }
    } else {
      tc_load_queries<T, D_>(p, w, TT, q_dst, q_full, lane);
    }
    qr.next(C::QST);
    for (int j = 0; j < w.nkt; ++j) {
      const int nb = min(8, (w.k1 - w.k0 - j * 128 + 15) >> 4);
      if (!mbar_wait(bar.k_empty(kr.st), kr.ph ^ 1, p.status)) return;
      tc_load<D_, false>(p, tk, k_s + kr.st * C::TILE, bar.k_full(kr.st), cur, key, nb, w.kvh, pol, lane, poison, seq);
      __syncwarp();  // (the item's mark comes before the V tile is announced, and so before every epilogue)
      kr.next(C::KST);
      if (!mbar_wait(bar.v_empty(vr.st), vr.ph ^ 1, p.status)) return;
      tc_load<D_, true>(p, tv, v_s + vr.st * C::TILE, bar.v_full(vr.st), cur, key, nb, w.kvh, pol, lane, poison, seq);
      vr.next(C::VST);
      if (j + 1 < w.nkt) cur = tc_block(p, w, btrow, j + 1, lane, key);
    }
  }
}

template <int D_>
__device__ void tc_mma(const MaskedParams& p, int TT, const TcBars& bar, uint32_t tmem, uint32_t q_s, uint32_t k_s,
                       uint32_t v_s, bool bf, TcRing& ring) {
  using C = TcCfg<D_>;
  const bool leader = elect_one();
  constexpr uint32_t REG = 128 * 128;  // one 64-element region of a 128-row operand
  const uint32_t idesc_s = umma_idesc_f16(bf, 128, 128, false, false);
  const uint32_t idesc_o = umma_idesc_f16(bf, 128, D_, false, true);
  Ring qr, kr, vr;
  int n_s[2] = {0, 0}, n_p[2] = {0, 0};
  uint32_t clean = 0;  // parity of each V stage's next masked tile
  auto wait_p = [&](int h) -> bool {
    if (!mbar_wait(bar.p_full(h), n_p[h] & 1, p.status)) return false;
    ++n_p[h];
    return true;
  };
  // warp-uniform bases; stages, halves and k-steps are offsets of the descriptors' address field
  tmem = __shfl_sync(0xffffffffu, tmem, 0);
  const uint64_t dq = umma_sdesc_sw128(__shfl_sync(0xffffffffu, q_s, 0), 16, 1024);
  const uint64_t dk = umma_sdesc_sw128(__shfl_sync(0xffffffffu, k_s, 0), 16, 1024);
  const uint64_t dv = umma_sdesc_sw128(__shfl_sync(0xffffffffu, v_s, 0), D_ == 64 ? REG : 2048, 1024);
  auto issue_pv = [&](int h, int vst, bool first) {
    tc_fence_after();
    const uint64_t b0 = dv + (uint64_t)(vst * (C::TILE >> 4));
    const uint32_t d = tmem + C::o_col(h), a0 = tmem + C::p_col(h);
    if (leader) {
      umma_f16_ts(d, a0, b0, idesc_o, first ? 0u : 1u);
#pragma unroll
      for (int kk = 1; kk < 8; ++kk) umma_f16_ts(d, a0 + kk * 8, b0 + (uint64_t)(kk * C::V_BLOCK >> 4), idesc_o, 1u);
      umma_commit(bar.o_done(h));
    }
    __syncwarp();
  };
  auto issue_s = [&](int h, int qh, int kst) {
    const uint64_t a0 = dq + (uint64_t)((qr.st * 2 + qh) * (C::TILE >> 4)), b0 = dk + (uint64_t)(kst * (C::TILE >> 4));
    const uint32_t d = tmem + C::s_col(h);
    if (leader) {
#pragma unroll
      for (int k = 0; k < D_ / 16; ++k) {
        const uint64_t off = (uint64_t)(((k >> 2) * REG + (k & 3) * 32) >> 4);
        umma_f16_ss(d, a0 + off, b0 + off, idesc_s, k > 0 ? 1u : 0u);
      }
      umma_commit(bar.s_full(h));
    }
    __syncwarp();
  };
  for (int slot; (slot = ring.next(p.status)) >= 0;) {
    const TcItem w = ring.item(slot);
    ring.release();
    if (w.bad) continue;
    // P V runs `lag` tiles behind S: one, or two where the halves take tiles in turn (a half's next S is then issued
    // while the other half's weights are still to come)
    const int lag = w.dup ? 2 : 1;
    int v1 = -1, v2 = -1;  // V stages of the last tile loaded and the one before
    auto values = [&](int j, int vst) -> bool {  // tile j's values may be used
      if (!w.masked(j)) return true;
      if (!mbar_wait(bar.v_clean(vst), clean >> vst & 1u, p.status)) return false;
      clean ^= 1u << vst;
      return true;
    };
    auto pv = [&](int j, int vst) -> bool {  // P V of tile j from V stage vst
      if (!values(j, vst)) return false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!w.active(h, j)) continue;
        if (!wait_p(h)) return false;
        issue_pv(h, vst, j < lag);  // (a half's first tile overwrites O_h)
      }
      return true;
    };
    if (!mbar_wait(bar.q_full(qr.st), qr.ph, p.status)) return;
    for (int j = 0; j < w.nkt; ++j) {
      if (!mbar_wait(bar.k_full(kr.st), kr.ph, p.status)) return;
      const int jp = j - lag, vst = lag == 1 ? v1 : v2;
      if (C::P_ALIAS) {
        // P_h sits in S_h: it is consumed before S_h is rewritten
        if (w.dup) {
          if (jp >= 0 && !pv(jp, vst)) return;
          tc_fence_after();
          issue_s(j & 1, 0, kr.st);
        } else {
          if (jp >= 0 && !values(jp, vst)) return;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h >= w.n_half) continue;
            if (jp >= 0) {
              if (!wait_p(h)) return;
              issue_pv(h, vst, jp == 0);
            }
            tc_fence_after();
            issue_s(h, h, kr.st);
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!w.active(h, j)) continue;
          if (!mbar_wait(bar.s_free(h), (n_s[h] & 1) ^ 1, p.status)) return;
          ++n_s[h];
          tc_fence_after();
          issue_s(h, w.dup ? 0 : h, kr.st);
        }
      }
      if (leader) umma_commit(bar.k_empty(kr.st));
      kr.next(C::KST);
      if (!C::P_ALIAS && jp >= 0 && !pv(jp, vst)) return;
      if (jp >= 0 && leader) umma_commit(bar.v_empty(vst));
      if (!mbar_wait(bar.v_full(vr.st), vr.ph, p.status)) return;
      v2 = v1;
      v1 = vr.st;
      vr.next(C::VST);
    }
    // every S of the item is issued: the Q stage is free once they complete
    if (leader) umma_commit(bar.q_empty(qr.st));
    qr.next(C::QST);
    if (lag == 2) {  // (such an item has two tiles or more)
      if (!pv(w.nkt - 2, v2)) return;
      if (leader) umma_commit(bar.v_empty(v2));
    }
    if (!pv(w.nkt - 1, v1)) return;
    if (leader) umma_commit(bar.v_empty(v1));
  }
}

// One row's attention over the item's keys in plain float32, one key at a
// time (an item whose values are not finite where some of its rows see them or
// whose blocks are not all there, a row without a sum of weights).
template <typename T, int D_>
__device__ __noinline__ void tc_row_again(const MaskedParams& p, const MaskedGroup g, int k0, int k1, int part, int kvh,
                                          int tok, int hd) {
  const VirtualKeys vk(p, g);
  const int* btrow = p.bt + (long long)g.slot * p.max_blocks;
  const int head = kvh * p.G + hd;
  const T* q = reinterpret_cast<const T*>(p.q) + (long long)(g.q_row0 + tok) * p.q_stride + (long long)head * D_;
  float acc[D_], m = -INFINITY, l = 0.f;
  for (int d = 0; d < D_; ++d) acc[d] = 0.f;
  for (int v = k0; v < k1; ++v) {
    const int key = vk.key(v);
    if (!sees(p, g, tok, key)) continue;
    const long long row = key_row(p, btrow, key);
    if (row < 0) continue;
    const long long off = (row * p.Hkv + kvh) * D_;
    const T* kr = reinterpret_cast<const T*>(p.kp) + off;
    const T* vr = reinterpret_cast<const T*>(p.vp) + off;
    float x = 0.f;
    for (int d = 0; d < D_; ++d) x = fmaf(Elem<T>::to_f(q[d]), Elem<T>::to_f(kr[d]), x);
    x *= p.scale_log2;
    const float mn = fmaxf(m, x), base = mn == -INFINITY ? 0.f : mn;
    const float a = ex2(m - base), e = ex2(x - base);
    m = mn;
    l = l * a + e;
    for (int d = 0; d < D_; ++d) acc[d] = fmaf(e, Elem<T>::to_f(vr[d]), acc[d] * a);
  }
  if (part >> 16 == 1) {
    const float inv = no_output(p, g, tok, l) ? kNaN : state_inverse(l);
    T* dst = reinterpret_cast<T*>(p.out) + (long long)(g.q_row0 + tok) * p.out_stride + (long long)head * D_;
    for (int d = 0; d < D_; ++d) dst[d] = Elem<T>::from_f(acc[d] * inv);
  } else if (float* rec = part_base(p, g, part & 0xffff, kvh)) {
    const int R = g.ntok * p.G, r = tok * p.G + hd;
    for (int d = 0; d < D_; ++d) rec[((d >> 2) * R + r) * 4 + (d & 3)] = acc[d];
    rec[(D_ / 4 * R + r) * 4] = m;
    rec[(D_ / 4 * R + r) * 4 + 1] = l;
  }
}

// The value warps: the rows of masked tiles, two a thread, zeroed when they
// are past the unit's keys or not finite; an item some row of which sees such
// a row is poisoned.
template <typename T, int D_>
__device__ void tc_values(const MaskedParams& p, const TcBars& bar, unsigned char* base, uint32_t v_s, TcRing& ring) {
  using C = TcCfg<D_>;
  constexpr uint32_t EX = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  const int lane = threadIdx.x & 31;
  volatile int* poison = reinterpret_cast<volatile int*>(base + kTcPoison);
  Ring vr;
  int seq = 0;
  for (int slot; (slot = ring.next(p.status)) >= 0; ring.release()) {
    const TcItem& w = ring.item(slot);
    if (w.bad) continue;
    ++seq;
    const int nkt = w.nkt;
    for (int j = 0; j < nkt; ++j, vr.next(C::VST)) {
      // (every tile is waited for and given back, so that these warps are never a whole turn of the ring away)
      if (!mbar_wait(bar.v_full(vr.st), vr.ph, p.status)) return;
      const bool masked = w.masked(j);
#pragma unroll 1
      for (int row = masked ? threadIdx.x & 63 : 128; row < 128; row += 64) {
        const uint32_t vs = v_s + vr.st * C::TILE + (row >> 4) * C::V_BLOCK + (row & 15) * 128;
        const int v = w.k0 + 128 * j + row;
        bool odd = v >= w.k1;
        if (!odd) {
#pragma unroll
          for (int c = 0; c < D_ / 8; ++c) {
            uint32_t e[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(e[0]), "=r"(e[1]), "=r"(e[2]), "=r"(e[3])
                         : "r"(vs + (c >> 3) * 2048 + (((c & 7) ^ (row & 7)) << 4)));
#pragma unroll
            for (int q = 0; q < 4; ++q) odd |= (e[q] & EX) == EX || ((e[q] >> 16) & EX) == EX;
          }
          if (odd && seen_by_any(p, w.g, w.key(v))) poison[seq & 7] = seq;
        }
        if (odd) {
#pragma unroll
          for (int c = 0; c < D_ / 8; ++c)
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vs + (c >> 3) * 2048 + ((c & 7) << 4)), "r"(0)
                         : "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
      }
      __syncwarp();
      if (lane == 0) {
        if (masked) mbar_arrive(bar.v_clean(vr.st));
        mbar_arrive(bar.v_empty(vr.st));
      }
    }
  }
}

template <typename T, int D_>
__device__ void tc_softmax(const MaskedParams& p, int TT, bool out16, const TcBars& bar, unsigned char* base,
                           uint32_t tmem, int h, TcRing& ring) {
  using C = TcCfg<D_>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = warp & 3, row = quad * 32 + lane;  // tensor-memory lanes of this warp: quad*32..
  const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
  const uint32_t s_addr = tmem + lane_addr + C::s_col(h), o_addr = tmem + lane_addr + C::o_col(h);
  const uint32_t p_addr = tmem + lane_addr + C::p_col(h);
  volatile int* poison = reinterpret_cast<volatile int*>(base + kTcPoison);  // [8]: item numbers, by their low bits
  float2* stats = reinterpret_cast<float2*>(base + kTcStats);  // half 1's (m, l) of a joined item
  int n_s = 0, n_o = 0, n_join = 0;
  const int tok0 = row / p.G, hd = row - tok0 * p.G;  // token of the half and query head of this row
  // a scale of 0 or less cannot follow the maximum and the mask: the scores are scaled before them then
  const float scale = p.scale_log2 > 0.f ? p.scale_log2 : 1.f;
  bool join_pending = false;  // half 1: its accumulator is still to be read by half 0
  int seq = 0;
  // The item itself stays in its slot of shared memory while the tiles run (its fields would cost the tile loop the
  // registers of the scores); what masked tiles and the epilogue need is read there again.
  for (int slot; (slot = ring.next(p.status)) >= 0; ring.release()) {
    int nkt, whole0, whole1;
    bool dup, valid;
    {
      const TcItem& w = ring.item(slot);
      if (w.bad) continue;
      ++seq;
      if (w.tiles(h) == 0) continue;
      nkt = w.nkt;
      whole0 = w.whole0;
      whole1 = w.whole1;
      dup = w.dup;
      valid = tok0 < TT && (dup ? 0 : h * TT) + tok0 < w.g.ntok;
    }
    float m = 0.f, l = 0.f;  // the reference of the exponents, and the sum of the weights
    bool none = true;        // no score of the row has had a place in a maximum yet
    int n = 0;  // tiles done
    for (int j = dup ? h : 0; j < nkt; j += dup ? 2 : 1, ++n) {
      if (!mbar_wait(bar.s_full(h), n_s & 1, p.status)) return;
      ++n_s;
      tc_fence_after();
      const bool masked = j < whole0 || j >= whole1;
      uint32_t x[128];
      float alpha = 1.f;
      uint64_t sum2[4];
      // the tile's scores into registers, unseen ones -inf
      auto scores = [&]() {
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(x + 32 * c));
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_reg_fence(*reinterpret_cast<uint32_t(*)[32]>(x + 32 * c));
        if (!C::P_ALIAS) {  // S_h is in registers: the next S_h may be computed
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar.s_free(h));
        }
        if (p.scale_log2 <= 0.f) {
#pragma unroll
          for (int i = 0; i < 128; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * p.scale_log2);
        }
        if (masked) {
          uint32_t bits[4] = {0u, 0u, 0u, 0u};
          if (valid) {
            row_bits(p, ring.item(slot), (dup ? 0 : h * TT) + tok0, j, bits);
          }
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (!(bits[i >> 5] >> (i & 31) & 1u)) x[i] = 0xff800000u;
        }
      };
      // weights against the reference m in the low half of x, and their sums
      auto weights = [&]() {
        const uint64_t sc2 = f2_pack(scale, scale), nb2 = f2_pack(-m, -m);
#pragma unroll
        for (int a = 0; a < 4; ++a) sum2[a] = 0ull;
#pragma unroll
        for (int i = 0; i < 128; i += 2) {
          const uint64_t y2 = f2_fma(f2_pack(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sc2, nb2);
          float y0, y1;
          f2_unpack(y2, y0, y1);
          const float p0 = ex2(y0), p1 = ex2(y1);
          sum2[(i >> 1) & 3] = f2_add(sum2[(i >> 1) & 3], f2_pack(p0, p1));
          x[i >> 1] = pack2<T>(p0, p1);
        }
      };
      // lazy rescaling: the reference moves only to a row's first seen scores, and when a score exceeds it by more
      // than 8 (weights stay below 2^8)
      {
        scores();
        float acc[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) acc[a] = fmaxf(__uint_as_float(x[a]), __uint_as_float(x[a + 8]));
#pragma unroll
        for (int i = 16; i < 128; i += 16)
#pragma unroll
          for (int a = 0; a < 8; ++a) acc[a] = fmax3(acc[a], __uint_as_float(x[i + a]), __uint_as_float(x[i + 8 + a]));
        const float mt = scale * fmaxf(fmaxf(fmaxf(acc[0], acc[1]), fmaxf(acc[2], acc[3])),
                                       fmaxf(fmaxf(acc[4], acc[5]), fmaxf(acc[6], acc[7])));
        if (none ? mt > -INFINITY : mt > m + 8.f) {
          if (!none) alpha = ex2(m - mt);
          m = mt;
          none = false;
        }
        weights();
      }
      if (n > 0) {  // O_h += P_h V of the half's tile before must be done before P_h or O_h change
        // (with P_h in S_h it was issued before this tile's S_h, which is complete)
        if (!C::P_ALIAS && !mbar_wait(bar.o_done(h), n_o & 1, p.status)) return;
        ++n_o;
        tc_fence_after();
      } else if (join_pending) {  // half 0 has read this half's last accumulator
        if (!mbar_wait(bar.join_empty(), (n_join - 1) & 1, p.status)) return;
        join_pending = false;
      }
      tmem_st32(p_addr, *reinterpret_cast<uint32_t(*)[32]>(x));
      tmem_st32(p_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(x + 32));
      if (n > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
        for (int c = 0; c < D_ / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
          tmem_reg_fence(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(o_addr + c * 32, o);
        }
      }
      float sa[8];
#pragma unroll
      for (int a = 0; a < 4; ++a) f2_unpack(sum2[a], sa[2 * a], sa[2 * a + 1]);
      l = l * alpha + (((sa[0] + sa[1]) + (sa[2] + sa[3])) + ((sa[4] + sa[5]) + (sa[6] + sa[7])));
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar.p_full(h));
    }
    if (!mbar_wait(bar.o_done(h), n_o & 1, p.status)) return;
    ++n_o;
    tc_fence_after();
    if (none) m = -INFINITY;
    const TcItem& w = ring.item(slot);
    const int tok = (dup ? 0 : h * TT) + tok0;
    float a0 = 1.f, a1 = 0.f;  // weights of this half's and half 1's accumulators
    if (w.dup) {
      ++n_join;
      if (h == 1) {
        stats[row] = make_float2(m, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar.join_full());
        join_pending = true;
        continue;
      }
      if (!mbar_wait(bar.join_full(), (n_join - 1) & 1, p.status)) return;
      tc_fence_after();
      const float2 other = stats[row];
      const float mn = fmaxf(m, other.x), b = mn == -INFINITY ? 0.f : mn;
      a0 = ex2(m - b);
      a1 = ex2(other.x - b);
      l = l * a0 + other.y * a1;
      m = mn;
    }
    const int n_parts = w.part >> 16, R = w.g.ntok * p.G, r = tok * p.G + hd;
    float4* rec = nullptr;
    // the row's place in out, in elements (-1: not a row)
    long long at = -1;
    if (n_parts == 1) {
      const float inv = state_inverse(l);
      a0 *= inv;
      a1 *= inv;
      if (valid) at = (long long)(w.g.q_row0 + tok) * p.out_stride + (long long)(w.kvh * p.G + hd) * D_;
    } else if (valid) {
      rec = reinterpret_cast<float4*>(part_base(p, w.g, w.part & 0xffff, w.kvh));
    }
#pragma unroll
    for (int c = 0; c < D_ / 64; ++c) {
      uint32_t o[64];
      tmem_ld32(o_addr + c * 64, *reinterpret_cast<uint32_t(*)[32]>(o));
      tmem_ld32(o_addr + c * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(o + 32));
      tmem_wait_ld();
      tmem_reg_fence(*reinterpret_cast<uint32_t(*)[32]>(o));
      tmem_reg_fence(*reinterpret_cast<uint32_t(*)[32]>(o + 32));
      if (w.dup) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t o1[32];
          tmem_ld32(o_addr - C::o_col(0) + C::o_col(1) + c * 64 + b * 32, o1);
          tmem_wait_ld();
          tmem_reg_fence(o1);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            o[32 * b + i] = __float_as_uint(fmaf(__uint_as_float(o1[i]), a1, __uint_as_float(o[32 * b + i]) * a0));
        }
      } else if (n_parts == 1) {
#pragma unroll
        for (int i = 0; i < 64; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a0);
      }
      if (n_parts > 1) {
        if (rec) {
#pragma unroll
          for (int i = 0; i < 16; ++i)  // lanes are rows: 512 contiguous bytes a store
            __stcg(rec + (c * 16 + i) * R + r, make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                          __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3])));
        }
        continue;
      }
      // eight lanes exchange 16-byte pieces (an 8 x 8 transpose in three steps), so that they store one row's 128
      // bytes together instead of a piece of eight rows each
      uint32_t v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = pack2<T>(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
#pragma unroll
      for (int st = 1; st < 8; st <<= 1) {
        const bool up = lane & st;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (q & st) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t &lo = v[4 * q + e], &hi = v[4 * (q ^ st) + e];
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, st);
            if (up)
              lo = got;
            else
              hi = got;
          }
        }
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const long long row_at = __shfl_sync(0xffffffffu, at, (lane & ~7) + q);
        if (row_at < 0) continue;
        T* d = reinterpret_cast<T*>(p.out) + row_at + c * 64 + (lane & 7) * 8;
        if (out16) {
          *reinterpret_cast<uint4*>(d) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            reinterpret_cast<unsigned short*>(d)[2 * e] = v[4 * q + e] & 0xffff;
            reinterpret_cast<unsigned short*>(d)[2 * e + 1] = v[4 * q + e] >> 16;
          }
        }
      }
    }
    if (rec) __stcg(reinterpret_cast<float2*>(rec + D_ / 4 * R + r), make_float2(m, l));
    tc_fence_before();
    if (w.dup) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar.join_empty());
    }
    __syncwarp();  // (eight lanes have stored a row together: before its own lane stores it again)
    // (l = 0: nothing seen, or 0 / 0)
    if (valid && (poison[seq & 7] == seq || (l == 0.f && n_parts == 1)))
      tc_row_again<T, D_>(p, w.g, w.k0, w.k1, w.part, w.kvh, tok, hd);
  }
}

template <typename T, int D_>
__global__ void __launch_bounds__(TcCfg<D_>::THREADS, 1)
    masked_tc_kernel(const MaskedParams p, int TT, int q_tma, int out16, const __grid_constant__ CUtensorMap tq,
                     const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv) {
  using C = TcCfg<D_>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t hdr = smem_u32(base);
  const TcBars bar(hdr);
  const int warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  if (threadIdx.x == 32) {
    tma_prefetch_map(&tk);
    tma_prefetch_map(&tv);
    if (q_tma) tma_prefetch_map(&tq);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::KST; ++s) {
      mbar_init(bar.k_full(s), 1);
      mbar_init(bar.k_empty(s), 1);
    }
    for (int s = 0; s < C::VST; ++s) {
      mbar_init(bar.v_full(s), 1);
      mbar_init(bar.v_empty(s), 1 + 2);  // P V's commit and the value warps
      mbar_init(bar.v_clean(s), 2);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(bar.s_full(h), 1);
      mbar_init(bar.s_free(h), 4);
      mbar_init(bar.p_full(h), 4);
      mbar_init(bar.o_done(h), 1);
    }
    for (int s = 0; s < C::QST; ++s) {
      mbar_init(bar.q_full(s), 1);
      mbar_init(bar.q_empty(s), 1);
    }
    for (int s = 0; s < kTcItemRing; ++s) {
      mbar_init(bar.item_full(s), 1);
      mbar_init(bar.item_empty(s), 1 + 2 + 4 * 2);  // the MMA, value and softmax warps
    }
    mbar_init(bar.join_full(), 4);
    mbar_init(bar.join_empty(), 4);
    fence_mbar_init();
    for (int i = 0; i < 8; ++i) reinterpret_cast<int*>(base + kTcPoison)[i] = 0;
  }
  if (warp == 1) tmem_alloc(hdr + kTcTmemPtr, C::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(base + kTcTmemPtr);
  const uint32_t q_s = hdr + C::Q_OFF, k_s = hdr + C::K_OFF, v_s = hdr + C::V_OFF;
  const int tasks = min(__ldg(p.counts + 1), p.max_items) * p.Hkv;
  TcRing ring(bar, base);
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_CTRL));
    if (warp == 0)
      tc_producer<T, D_>(p, TT, q_tma, &tq, &tk, &tv, bar, base, q_s, k_s, v_s, tasks, ring);
    else if (warp == 1)
      tc_mma<D_>(p, TT, bar, tmem, q_s, k_s, v_s, std::is_same<T, __nv_bfloat16>::value, ring);
    else
      tc_values<T, D_>(p, bar, base, v_s, ring);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SOFTMAX));
    tc_softmax<T, D_>(p, TT, out16, bar, base, tmem, (warp - 4) >> 2, ring);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::TMEM_COLS);
  // every ticket of every CTA is taken when the last CTA is out
  if (threadIdx.x == 0 && atomicAdd(p.queue + 3, 1) == (int)gridDim.x - 1) {
    p.queue[2] = 0;
    p.queue[3] = 0;
    __threadfence();
  }
}

// 256 rows of whole tokens, for the shapes whose small groups the tensor-map kernel takes.
int masked_tc_rows(int dtype, int Hq, int Hkv, int D, int bs) {
  if (!masked_tma_rows(dtype, Hq, Hkv, D, bs)) return 0;
  const int G = Hq / Hkv;
  return 2 * (128 / G) * G;
}

template <typename T, int D_>
static int launch_tc(const MaskedParams& p, int TT, int q_tma, int out16, const CUtensorMap& tq, const CUtensorMap& tk,
                     const CUtensorMap& tv, cudaStream_t st, const char* what) {
  using C = TcCfg<D_>;
  auto kern = masked_tc_kernel<T, D_>;
  cudaError_t e = prepare_launch(reinterpret_cast<const void*>(kern), (int)C::SMEM, C::THREADS, nullptr);
  if (e != cudaSuccess) return fail(NF_ECUDA, "%s: smem attribute: %s", what, cudaGetErrorString(e));
  static int regs = -1;  // a property of the binary, queried once
  if (regs < 0) {
    cudaFuncAttributes fa;
    regs = cudaFuncGetAttributes(&fa, kern) == cudaSuccess ? fa.numRegs : 0;
  }
  if (C::REGS_CTRL * 128 + C::REGS_SOFTMAX * 256 > regs * C::THREADS)
    return fail(NF_EUNSUPPORTED, "%s: kernel built with %d registers per thread, the warpgroup split needs 168", what, regs);
  long long grid = (long long)p.max_items * p.Hkv;
  if (grid > sm_count()) grid = sm_count();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, p, TT, q_tma, out16, tq, tk, tv);
  if (e != cudaSuccess) return fail(NF_ECUDA, "%s: launch: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

int launch_masked_tc(const MaskedParams& p, int dtype, void* stream, const char* what) {
  if (!masked_tc_rows(dtype, p.Hq, p.Hkv, p.D, p.bs))
    return fail(NF_EUNSUPPORTED, "%s: no tensor-core items for this shape", what);
  if ((reinterpret_cast<uintptr_t>(p.kp) | reinterpret_cast<uintptr_t>(p.vp)) & 15)
    return fail(NF_EINVAL, "%s: pools must be 16-byte aligned", what);
  if ((long long)p.max_items * p.Hkv > INT32_MAX) return fail(NF_EINVAL, "%s: too many items", what);
  const int TT = 128 / p.G;
  const int q_tma = reinterpret_cast<uintptr_t>(p.q) % 16 == 0 && p.q_stride % 8 == 0 && p.q_stride > 0;
  const int out16 = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_stride % 8 == 0;
  CUtensorMap tq, tk, tv;
  if (!encode_pool_map(&tk, p.kp, dtype, p.D, p.Hkv, p.bs, p.num_blocks, 1, false) ||
      !encode_pool_map(&tv, p.vp, dtype, p.D, p.Hkv, p.bs, p.num_blocks, 1, p.D == 128) ||
      (q_tma && !encode_rows_map(&tq, p.q, dtype, p.D, p.Hq, p.rows, p.q_stride, p.G, TT)))
    return fail(NF_ECUDA, "%s: tensor map encoding failed", what);
  if (!q_tma) tq = tk;  // (not used)
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == NF_BF16)
    return p.D == 64 ? launch_tc<__nv_bfloat16, 64>(p, TT, q_tma, out16, tq, tk, tv, st, what)
                     : launch_tc<__nv_bfloat16, 128>(p, TT, q_tma, out16, tq, tk, tv, st, what);
  return p.D == 64 ? launch_tc<__half, 64>(p, TT, q_tma, out16, tq, tk, tv, st, what)
                   : launch_tc<__half, 128>(p, TT, q_tma, out16, tq, tk, tv, st, what);
}

}  // namespace nf
