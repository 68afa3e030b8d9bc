// Windowed and tree attention: the per-warp kernel for every type and shape,
// the merge of split-K parts and the entry points.  See nf_masked.cuh for the
// operators' definition and the work records.
#include "nf_internal.h"
#include "nf_masked.cuh"

namespace nf {

// Columns (token, query head of the KV head) that one CTA task carries.
constexpr int kVecCols = 4;
// Query rows of a group of these kernels (at least one token), and the most of
// a step's largest group that go to the kernel of few columns: above, tiles of
// 32 columns read each key once for them.
constexpr int kVecRows = 32;
constexpr int kVecMost = 8;
constexpr int kVecWarps = 8;

template <typename T, int VW> struct VecLoad;
template <> struct VecLoad<float, 4> {
  static __device__ __forceinline__ void load(const float* p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  }
};
template <typename H> struct VecLoad<H, 8> {
  static __device__ __forceinline__ void load(const H* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const H* h = reinterpret_cast<const H*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<H>::to_f(h[i]);
  }
};
template <typename H> struct VecLoad<H, 1> {
  static __device__ __forceinline__ void load(const H* p, float (&x)[1]) { x[0] = Elem<H>::to_f(*p); }
};

// A CTA computes C columns of one (unit, KV head): its warps take the unit's
// keys in turn, KPW at a time a step (LPK lanes hold a key's row, VW elements
// a load, EV loads; every lane group has a running maximum, sum and output of
// its own), and are joined through shared memory at the end.  Bound by the
// key and value bytes (column chunks of a group read them again, from L2) and,
// for short key ranges, by the latency of the dependent loads: eight warps on
// a unit make that two or three steps, and one unit a sequence needs no merge
// (8 float32 decodes of 12 heads over 130 keys: 7.6 us; 41 with a warp a unit
// of 64 keys and a merge.  64 float32 decodes with full contexts, 0.9 GB:
// 164 us, 86 % of the copy bandwidth.)
template <typename T, int VW, int LPK, int EV, int C>
__global__ void __launch_bounds__(kVecWarps * 32, C == 1 ? 3 : 2) masked_vec_kernel(const MaskedParams p) {
  constexpr int KPW = 32 / LPK;  // keys per step of the warp
  constexpr int U = EV * VW >= 8 ? 2 : 4;  // steps in flight
  constexpr int E = EV * VW;
  extern __shared__ float joined[];  // [kVecWarps][C][D + 2]
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, li = lane % LPK, lg = lane / LPK;
  const int n_units = min(__ldg(p.counts + 3), p.max_units);
  pdl_wait();
  const T* q = reinterpret_cast<const T*>(p.q);
  const T* kp = reinterpret_cast<const T*>(p.kp);
  const T* vp = reinterpret_cast<const T*>(p.vp);
  const long long row_elems = (long long)p.Hkv * p.D;
  const int chunks = (p.unit_tokens * p.G + C - 1) / C;  // of the largest group; a smaller one's last tasks are empty
  const long long tasks = (long long)n_units * p.Hkv * chunks;
  for (long long task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int u = (int)(task / (p.Hkv * chunks)), rest = (int)(task - (long long)u * p.Hkv * chunks);
    const int kvh = rest / chunks, c0 = (rest - kvh * chunks) * C;
    MaskedGroup g;
    const int4 un = load_record(p.units, u, g);
    if (!unit_ok(p, un, g)) {
      if (threadIdx.x == 0) atomicOr(p.status, NF_STATUS_BAD_SLOT);
      continue;
    }
    const int cols = g.ntok * p.G;
    if (c0 >= cols) continue;
    const VirtualKeys vk(p, g);
    const int* btrow = p.bt + (long long)g.slot * p.max_blocks;
    const int v1 = min(un.y, vk.end);
    float qr[C][E];
    int tok[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = min(c0 + c, cols - 1);
      tok[c] = col / p.G;
      const T* qrow = q + (long long)(g.q_row0 + tok[c]) * p.q_stride +
                      (long long)(kvh * p.G + (col - tok[c] * p.G)) * p.D;
#pragma unroll
      for (int v = 0; v < EV; ++v) {
        const int e = (v * LPK + li) * VW;
#pragma unroll
        for (int i = 0; i < VW; ++i)  // queries may start at any element of their row's allocation: element loads
          qr[c][v * VW + i] = e < p.D ? Elem<T>::to_f(qrow[e + i]) * p.scale_log2 : 0.f;
      }
    }
    float m[C], l[C], acc[C][E];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      m[c] = -INFINITY;
      l[c] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[c][e] = 0.f;
    }
    for (int v0 = un.x + warp * (KPW * U); v0 < v1; v0 += kVecWarps * KPW * U) {
      float kx[U][E], vx[U][E];
      int key[U];
      long long row[U];
      // every load of the U steps first
#pragma unroll
      for (int s = 0; s < U; ++s) {
        const int v = v0 + s * KPW + lg;
        key[s] = v < v1 ? vk.key(v) : -1;
        row[s] = key[s] >= 0 ? key_row(p, btrow, key[s]) : -1;
        if (row[s] < 0) key[s] = -1;
      }
#pragma unroll
      for (int s = 0; s < U; ++s)
#pragma unroll
        for (int w = 0; w < EV; ++w) {
          const int e = (w * LPK + li) * VW;
          float a[VW], b[VW];
#pragma unroll
          for (int i = 0; i < VW; ++i) a[i] = b[i] = 0.f;
          if (row[s] >= 0 && e < p.D) {
            const long long off = row[s] * row_elems + (long long)kvh * p.D + e;
            VecLoad<T, VW>::load(kp + off, a);
            VecLoad<T, VW>::load(vp + off, b);
          }
#pragma unroll
          for (int i = 0; i < VW; ++i) {
            kx[s][w * VW + i] = a[i];
            vx[s][w * VW + i] = b[i];
          }
        }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float x[U];
        unsigned vis = 0;  // keys of this column: the others are left out, whatever their value rows hold
        float mn = m[c];
#pragma unroll
        for (int s = 0; s < U; ++s) {
          float d = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) d = fmaf(qr[c][e], kx[s][e], d);
#pragma unroll
          for (int o = LPK / 2; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
          if (key[s] >= 0 && sees(p, g, tok[c], key[s])) {
            vis |= 1u << s;
            mn = fmaxf(mn, d);
          }
          x[s] = d;
        }
        const float base = mn == -INFINITY ? 0.f : mn;
        const float al = ex2(m[c] - base);
        m[c] = mn;
        l[c] *= al;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[c][e] *= al;
#pragma unroll
        for (int s = 0; s < U; ++s) {
          if (vis >> s & 1u) {
            const float w = ex2(x[s] - base);
            l[c] += w;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[c][e] = fmaf(w, vx[s][e], acc[c][e]);
          }
        }
      }
    }
    // join the lane groups, then the warps
    const int DJ = p.D + 2;
    __syncthreads();  // (the task before has read the joined states)
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int o = LPK; o < 32; o <<= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m[c], o), lo = __shfl_xor_sync(0xffffffffu, l[c], o);
        const float mn = fmaxf(m[c], mo), base = mn == -INFINITY ? 0.f : mn;
        const float a = ex2(m[c] - base), b = ex2(mo - base);
        l[c] = l[c] * a + lo * b;
#pragma unroll
        for (int e = 0; e < E; ++e)
          acc[c][e] = acc[c][e] * a + __shfl_xor_sync(0xffffffffu, acc[c][e], o) * b;
        m[c] = mn;
      }
      if (lg != 0) continue;
      float* st = joined + (warp * C + c) * DJ;
#pragma unroll
      for (int v = 0; v < EV; ++v) {
        const int e = (v * LPK + li) * VW;
        if (e < p.D)
#pragma unroll
          for (int i = 0; i < VW; ++i) st[e + i] = acc[c][v * VW + i];
      }
      if (li == 0) {
        st[p.D] = m[c];
        st[p.D + 1] = l[c];
      }
    }
    __syncthreads();
    const int part = un.z & 0xffff, n_parts = un.z >> 16;
    float* rec = n_parts > 1 ? part_base(p, g, part, kvh) : nullptr;
    const int n = min(C, cols - c0) * p.D;
    for (int i = threadIdx.x; i < n; i += kVecWarps * 32) {
      const int c = i / p.D, e = i - c * p.D, col = c0 + c;
      float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
      for (int w = 0; w < kVecWarps; ++w) M = fmaxf(M, joined[(w * C + c) * DJ + p.D]);
      const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int w = 0; w < kVecWarps; ++w) {
        const float* st = joined + (w * C + c) * DJ;
        const float f = ex2(st[p.D] - base);
        A = fmaf(st[e], f, A);
        L = fmaf(st[p.D + 1], f, L);
      }
      if (n_parts == 1) {
        const int t = col / p.G, head = kvh * p.G + (col - t * p.G);
        T* dst = reinterpret_cast<T*>(p.out) + (long long)(g.q_row0 + t) * p.out_stride + (long long)head * p.D + e;
        *dst = Elem<T>::from_f(A * state_inverse(L));
        if (no_output(p, g, t, L)) *dst = Elem<T>::from_f(kNaN);
      } else if (rec) {
        float* r = rec + (long long)col * p.DP;
        r[e] = A;
        if (e == 0) *reinterpret_cast<float2*>(r + p.DP - 4) = make_float2(M, L);
      }
    }
  }
}

// Groups of many columns of the same types and shapes: a CTA takes 32 columns
// of one (unit, KV head), four a warp, and walks the unit's keys 32 at a time,
// K and V staged in shared memory as float32 (the next tile's rows travel
// through registers meanwhile).  Scores with a key a lane (no sums across
// lanes; rows padded so that the eight lanes of a 16-byte read hit distinct
// banks), value sums with an element a lane.  Bound by instructions (about
// 1,150 a warp and tile for 512 FMAs at head_dim 64): 8 float32 chunks of 200
// tokens, 12 heads and a window of 256 keys 129 us, with four columns a CTA 294;
// 25 trees of 16 tokens on 500 to 4,000 keys, 12 heads, 308 us, on 4,000 515.
// D <= 32 ND; two CTAs an SM up to 128 (in 128 registers: 6 trees of 20 tokens on
// 500 to 2,000 keys, 8 float32 heads of 128, 77 to 82 us; one CTA took a third more).
template <typename T, int ND, bool VEC>
__global__ void __launch_bounds__(256, ND <= 4 ? 2 : 1) masked_tile_kernel(const MaskedParams p) {
  constexpr int VW = sizeof(T) == 4 ? 4 : 8;
  extern __shared__ float4 tile_smem[];
  const int D4 = (p.D + 3) >> 2, KP = D4 + 1;  // float4s of a row, and of a padded K row
  float4* ks = tile_smem;             // [32][KP]
  float4* vs = ks + 32 * KP;          // [32][D4]
  float4* qs = vs + 32 * D4;          // [32][D4]
  float4* ps = qs + 32 * D4;          // [8 warps][32 keys]: four columns' weights
  // the last fetched tiles (even, odd) with rows in a block that is not there
  volatile int* missing = reinterpret_cast<volatile int*>(ps + 8 * 32);
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_units = min(__ldg(p.counts + 3), p.max_units);
  pdl_wait();
  const int blocks = (p.unit_tokens * p.G + 31) >> 5;
  const long long tasks = (long long)n_units * p.Hkv * blocks, row_elems = (long long)p.Hkv * p.D;
  for (long long task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int u = (int)(task / (p.Hkv * blocks)), rest = (int)(task - (long long)u * p.Hkv * blocks);
    const int kvh = rest / blocks, c0 = (rest - kvh * blocks) * 32;
    MaskedGroup g;
    const int4 un = load_record(p.units, u, g);
    if (!unit_ok(p, un, g)) {
      if (threadIdx.x == 0) atomicOr(p.status, NF_STATUS_BAD_SLOT);
      continue;
    }
    const int cols = g.ntok * p.G;
    if (c0 >= cols) continue;
    const VirtualKeys vk(p, g);
    const int* btrow = p.bt + (long long)g.slot * p.max_blocks;
    const int v1 = min(un.y, vk.end);
    const T* kp = reinterpret_cast<const T*>(p.kp) + (long long)kvh * p.D;
    const T* vp = reinterpret_cast<const T*>(p.vp) + (long long)kvh * p.D;
    __syncthreads();  // (the task before is done with the shared tiles)
    for (int i = threadIdx.x; i < 32 * D4 * 4; i += 256) {
      const int c = i / (D4 * 4), e = i - c * (D4 * 4), col = c0 + c;
      float x = 0.f;
      if (col < cols && e < p.D) {
        const int tok = col / p.G;
        x = Elem<T>::to_f(reinterpret_cast<const T*>(p.q)[(long long)(g.q_row0 + tok) * p.q_stride +
                                                         (long long)(kvh * p.G + col - tok * p.G) * p.D + e]);
      }
      reinterpret_cast<float*>(qs)[i] = x * p.scale_log2;
    }
    // this warp's columns; the tile after the one at work in registers
    const int w0 = c0 + 4 * warp;
    const bool busy = w0 < cols;
    int tok[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) tok[c] = min(w0 + c, cols - 1) / p.G;
    float m[4], l[4], o[4][ND];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      m[c] = -INFINITY;
      l[c] = 0.f;
#pragma unroll
      for (int i = 0; i < ND; ++i) o[c][i] = 0.f;
    }
    float4 kr[ND], vr[ND];
    auto fetch = [&](int v0) {
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int f = i * 256 + threadIdx.x, r = f / D4, e = (f - r * D4) * 4, v = v0 + r;
        kr[i] = vr[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r >= 32 || v >= v1) continue;
        const long long row = key_row(p, btrow, vk.key(v));
        if (row < 0) {
          missing[v0 >> 5 & 1] = v0;
          continue;
        }
        const T* a = kp + row * row_elems + e;
        const T* b = vp + row * row_elems + e;
        if constexpr (VEC && VW == 4) {
          kr[i] = *reinterpret_cast<const float4*>(a);
          vr[i] = *reinterpret_cast<const float4*>(b);
        } else if constexpr (VEC) {
          const uint2 x = *reinterpret_cast<const uint2*>(a), y = *reinterpret_cast<const uint2*>(b);
          const T* h = reinterpret_cast<const T*>(&x);
          const T* n = reinterpret_cast<const T*>(&y);
          kr[i] = make_float4(Elem<T>::to_f(h[0]), Elem<T>::to_f(h[1]), Elem<T>::to_f(h[2]), Elem<T>::to_f(h[3]));
          vr[i] = make_float4(Elem<T>::to_f(n[0]), Elem<T>::to_f(n[1]), Elem<T>::to_f(n[2]), Elem<T>::to_f(n[3]));
        } else {
          float x[4], y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[j] = e + j < p.D ? Elem<T>::to_f(a[j]) : 0.f;
            y[j] = e + j < p.D ? Elem<T>::to_f(b[j]) : 0.f;
          }
          kr[i] = make_float4(x[0], x[1], x[2], x[3]);
          vr[i] = make_float4(y[0], y[1], y[2], y[3]);
        }
      }
    };
    fetch(un.x);
    for (int v0 = un.x; v0 < v1; v0 += 32) {
      __syncthreads();  // the tile before is done with (and, first, the queries are in place)
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int f = i * 256 + threadIdx.x, r = f / D4, c = f - r * D4;
        if (r < 32) {
          ks[r * KP + c] = kr[i];
          vs[r * D4 + c] = vr[i];
        }
      }
      __syncthreads();
      if (v0 + 32 < v1) fetch(v0 + 32);
      if (!busy) continue;
      // scores: this lane's key against the warp's four columns
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      const float4* q = qs + 4 * warp * D4;
#pragma unroll 4
      for (int e = 0; e < D4; ++e) {
        const float4 k = ks[lane * KP + e];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 x = q[c * D4 + e];
          s[c] = fmaf(k.x, x.x, fmaf(k.y, x.y, fmaf(k.z, x.z, fmaf(k.w, x.w, s[c]))));
        }
      }
      const int v = v0 + lane, key = vk.key(v);
      const bool there = v < v1 && (missing[v0 >> 5 & 1] != v0 || key_row(p, btrow, key) >= 0);
      unsigned unseen = 0;  // columns that do not see the key
      float4 w;
      float* wp = reinterpret_cast<float*>(&w);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool seen = there && sees(p, g, tok[c], key);
        if (!seen) unseen |= 1u << c;
        float top = seen ? s[c] : -INFINITY;
        const float x = top;
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float mn = fmaxf(m[c], top), base = mn == -INFINITY ? 0.f : mn, al = ex2(m[c] - base);
        m[c] = mn;
        wp[c] = ex2(x - base);
        l[c] = l[c] * al + wp[c];
#pragma unroll
        for (int i = 0; i < ND; ++i) o[c][i] *= al;
      }
      // -0 for a key that is not seen: a seen one's weight may have underflowed to 0
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (unseen >> c & 1u) wp[c] = -0.f;
      ps[warp * 32 + lane] = w;
      __syncwarp();
      const float* vf = reinterpret_cast<const float*>(vs) + lane;
      if (__all_sync(0xffffffffu, unseen == 0)) {
#pragma unroll 4
        for (int k = 0; k < 32; ++k) {
          const float4 x = ps[warp * 32 + k];
#pragma unroll
          for (int i = 0; i < ND; ++i) {
            const float y = 32 * i + lane < p.D ? vf[k * D4 * 4 + 32 * i] : 0.f;
            o[0][i] = fmaf(x.x, y, o[0][i]);
            o[1][i] = fmaf(x.y, y, o[1][i]);
            o[2][i] = fmaf(x.z, y, o[2][i]);
            o[3][i] = fmaf(x.w, y, o[3][i]);
          }
        }
      } else {  // keys that a column does not see are left out, whatever their value rows hold
        constexpr unsigned kUnseen = 0x80000000u;
        for (int k = 0; k < 32; ++k) {
          const float4 x = ps[warp * 32 + k];
#pragma unroll
          for (int i = 0; i < ND; ++i) {
            const float y = 32 * i + lane < p.D ? vf[k * D4 * 4 + 32 * i] : 0.f;
            if (__float_as_uint(x.x) != kUnseen) o[0][i] = fmaf(x.x, y, o[0][i]);
            if (__float_as_uint(x.y) != kUnseen) o[1][i] = fmaf(x.y, y, o[1][i]);
            if (__float_as_uint(x.z) != kUnseen) o[2][i] = fmaf(x.z, y, o[2][i]);
            if (__float_as_uint(x.w) != kUnseen) o[3][i] = fmaf(x.w, y, o[3][i]);
          }
        }
      }
      __syncwarp();
    }
    if (!busy) continue;
    const int part = un.z & 0xffff, n_parts = un.z >> 16;
    float* rec = n_parts > 1 ? part_base(p, g, part, kvh) : nullptr;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float sum = l[c];
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const int col = w0 + c;
      if (col >= cols) continue;
      if (n_parts == 1) {
        const float inv = state_inverse(sum);
        T* dst = reinterpret_cast<T*>(p.out) + (long long)(g.q_row0 + tok[c]) * p.out_stride +
                 (long long)(kvh * p.G + col - tok[c] * p.G) * p.D;
#pragma unroll
        for (int i = 0; i < ND; ++i)
          if (32 * i + lane < p.D) dst[32 * i + lane] = Elem<T>::from_f(o[c][i] * inv);
        if (no_output(p, g, tok[c], sum))
          for (int e = lane; e < p.D; e += 32) dst[e] = Elem<T>::from_f(kNaN);
      } else if (rec) {
        float* r = rec + (long long)col * p.DP;
#pragma unroll
        for (int i = 0; i < ND; ++i)
          if (32 * i + lane < p.D) r[32 * i + lane] = o[c][i];
        if (lane == 0) *reinterpret_cast<float2*>(r + p.DP - 4) = make_float2(m[c], sum);
      }
    }
  }
}

// Merge of split-K parts: out = sum_j 2^(m_j - M) acc_j / sum_j 2^(m_j - M)
// l_j, always in the order of the parts.  A warp takes two rows of one
// (group, KV head): a lane holds a float4 of one of them, so a load is whole
// 32-byte sectors, and goes over the parts PB at a time with a running maximum
// (one round trip to L2 per PB parts).  A merge record covers four rows.  WAYS
// warps share the parts of a task (joined through shared memory): 48 parts of a
// long context would be twelve round trips for one.
template <typename T, int WAYS>
__global__ void __launch_bounds__(256, 4) masked_merge_kernel(const MaskedParams p) {
  constexpr int PB = 4, PER = 8 / WAYS;  // tasks a CTA
  __shared__ float4 join_a[WAYS > 1 ? 8 : 1][32];
  __shared__ float2 join_s[WAYS > 1 ? 8 : 1][32];
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, way = warp % WAYS;
  const int n = min(__ldg(p.counts + 2), p.max_merge);
  const int D4 = p.DP / 4 - 1;
  const long long tasks = (long long)n * p.Hkv * 2;
  // the first task's record is not of the launch before this one: it is read while that one ends
  MaskedGroup g;
  long long task = (long long)blockIdx.x * PER + warp / WAYS;
  int4 mr = load_record(p.merge, (int)min(task / (p.Hkv * 2), (long long)p.max_merge - 1), g);
  const long long first = task;
  pdl_wait();
  // (a CTA's warps go through the loop together: they join inside)
  for (; task - warp / WAYS < tasks; task += (long long)gridDim.x * PER) {
    const int i = (int)(task / (p.Hkv * 2)), rest = (int)(task - (long long)i * p.Hkv * 2), kvh = rest >> 1;
    if (task != first && task < tasks) mr = load_record(p.merge, i, g);
    bool ok = task < tasks;
    if (ok && (!group_ok(p, g) || mr.x <= 0 || mr.y < 0)) {
      if (lane == 0 && way == 0) atomicOr(p.status, NF_STATUS_UNIT_OVERFLOW);
      ok = false;
    }
    const int R = g.ntok * p.G, row = mr.y + 2 * (rest & 1) + (lane & 1);
    const float4* base = nullptr;
    // float4 c of the row at c * cs + at, and (m, l) as float4 D4
    const int cs = mr.z ? R : 1, at = mr.z ? row : row * (D4 + 1);
    if (ok && row < R && part_base(p, g, mr.x - 1, kvh))
      base = reinterpret_cast<const float4*>(part_base(p, g, 0, kvh)) + at;
    const long long step = (long long)g.ntok * p.Hq * (D4 + 1);  // float4s between consecutive parts
    for (int c0 = 0; c0 < D4; c0 += 16) {
      const int c = c0 + (lane >> 1);
      float M = -INFINITY, L = 0.f;
      float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
      if (base && c < D4)
        for (int j = way * PB; j < mr.x; j += WAYS * PB) {
          float4 x[PB];
          float2 ml[PB];
#pragma unroll
          for (int u = 0; u < PB; ++u)
            if (j + u < mr.x) {
              const float4* pj = base + (j + u) * step;
              ml[u] = __ldcg(reinterpret_cast<const float2*>(pj + D4 * cs));
              x[u] = __ldcg(pj + c * cs);
            } else {
              ml[u] = make_float2(-INFINITY, 0.f);
            }
          float nm = M;
#pragma unroll
          for (int u = 0; u < PB; ++u) nm = fmaxf(nm, ml[u].x);
          const float b = nm == -INFINITY ? 0.f : nm, sc = ex2(M - b);
          A.x *= sc; A.y *= sc; A.z *= sc; A.w *= sc; L *= sc;
#pragma unroll
          for (int u = 0; u < PB; ++u)
            if (ml[u].y != 0.f) {  // (0: no part, or one without seen keys)
              const float w = ex2(ml[u].x - b);
              A.x = fmaf(x[u].x, w, A.x); A.y = fmaf(x[u].y, w, A.y);
              A.z = fmaf(x[u].z, w, A.z); A.w = fmaf(x[u].w, w, A.w);
              L = fmaf(ml[u].y, w, L);
            }
          M = nm;
        }
      if constexpr (WAYS > 1) {
        __syncthreads();  // (the join before has been read)
        join_a[warp][lane] = A;
        join_s[warp][lane] = make_float2(M, L);
        __syncthreads();
        if (way == 0) {
          float nm = M;
#pragma unroll
          for (int w = 1; w < WAYS; ++w) nm = fmaxf(nm, join_s[warp + w][lane].x);
          const float b = nm == -INFINITY ? 0.f : nm, f0 = ex2(M - b);
          A.x *= f0; A.y *= f0; A.z *= f0; A.w *= f0; L *= f0;
#pragma unroll
          for (int w = 1; w < WAYS; ++w) {
            const float2 s = join_s[warp + w][lane];
            const float4 x = join_a[warp + w][lane];
            const float f = ex2(s.x - b);
            A.x = fmaf(x.x, f, A.x); A.y = fmaf(x.y, f, A.y); A.z = fmaf(x.z, f, A.z); A.w = fmaf(x.w, f, A.w);
            L = fmaf(s.y, f, L);
          }
        }
      }
      if (way != 0 || !base || c >= D4) continue;
      const int tok = row / p.G;
      const float inv = state_inverse(L);
      const float o[4] = {A.x * inv, A.y * inv, A.z * inv, A.w * inv};
      T* d = reinterpret_cast<T*>(p.out) + (long long)(g.q_row0 + tok) * p.out_stride +
             (long long)(kvh * p.G + row - tok * p.G) * p.D + 4 * c;
      if (sizeof(T) == 2 && 4 * c + 4 <= p.D && (reinterpret_cast<uintptr_t>(d) & 7) == 0) {
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint2*>(d) = make_uint2(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * c + e < p.D) d[e] = Elem<T>::from_f(o[e]);
      }
      if (no_output(p, g, tok, L))
        for (int e = 0; e < 4 && 4 * c + e < p.D; ++e) d[e] = Elem<T>::from_f(kNaN);
    }
  }
}

// Launch with programmatic stream serialization (the kernel waits for the
// one before it ahead of its first read of what that writes).
template <typename K>
static int launch_masked(K kern, long long blocks, int threads, cudaStream_t st, const MaskedParams& p,
                         const char* what, int smem = 0) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks < 1 ? 1 : blocks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return fail(NF_ECUDA, "%s: launch: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

template <typename T>
static int launch_merge(const MaskedParams& p, int max_parts, cudaStream_t st, const char* what) {
  // several warps a task where there are few tasks with many parts; with many tasks the loads in flight are enough
  const long long tasks = (long long)p.max_merge * p.Hkv * 2, cap = (long long)sm_count() * 8;
  const int ways = max_parts <= 8 || tasks > 2 * cap ? 1 : max_parts <= 16 ? 2 : 8;
  const long long want = (tasks * ways + 7) / 8;
  const long long blocks = want < cap ? want : cap;
  if (ways == 1) return launch_masked(masked_merge_kernel<T, 1>, blocks, 256, st, p, what);
  if (ways == 2) return launch_masked(masked_merge_kernel<T, 2>, blocks, 256, st, p, what);
  return launch_masked(masked_merge_kernel<T, 8>, blocks, 256, st, p, what);
}

template <typename T, int VW, int LPK, int EV>
static int launch_vec(const MaskedParams& p, cudaStream_t st, const char* what) {
  // one column where no group has more (decodes of a model without grouped heads), else four
  const bool one = p.unit_tokens * p.G == 1;
  const int C = one ? 1 : kVecCols;
  long long blocks = (long long)p.max_units * p.Hkv * ((p.unit_tokens * p.G + C - 1) / C);
  const long long cap = (long long)sm_count() * 8;
  if (blocks > cap) blocks = cap;
  const int smem = kVecWarps * C * (p.D + 2) * 4;  // 32 KB at most
  return one ? launch_masked(masked_vec_kernel<T, VW, LPK, EV, 1>, blocks, kVecWarps * 32, st, p, what, smem)
             : launch_masked(masked_vec_kernel<T, VW, LPK, EV, kVecCols>, blocks, kVecWarps * 32, st, p, what, smem);
}

template <typename T, int ND, bool VEC>
static int launch_tile(const MaskedParams& p, cudaStream_t st, const char* what) {
  const int D4 = (p.D + 3) / 4, smem = (32 * (D4 + 1) + 64 * D4 + 256 + 1) * 16;
  auto kern = masked_tile_kernel<T, ND, VEC>;
  const cudaError_t e = prepare_launch(reinterpret_cast<const void*>(kern), smem, 256, nullptr);
  if (e != cudaSuccess) return fail(NF_ECUDA, "%s: smem attribute: %s", what, cudaGetErrorString(e));
  long long blocks = (long long)p.max_units * p.Hkv * ((p.unit_tokens * p.G + 31) / 32);
  const long long cap = (long long)sm_count() * 8;
  if (blocks > cap) blocks = cap;
  return launch_masked(kern, blocks, 256, st, p, what, smem);
}

template <typename T, bool VEC>
static int dispatch_tile(const MaskedParams& p, cudaStream_t st, const char* what) {
  if (p.D <= 32) return launch_tile<T, 1, VEC>(p, st, what);
  if (p.D <= 64) return launch_tile<T, 2, VEC>(p, st, what);
  if (p.D <= 96) return launch_tile<T, 3, VEC>(p, st, what);
  if (p.D <= 128) return launch_tile<T, 4, VEC>(p, st, what);
  return launch_tile<T, 8, VEC>(p, st, what);
}

template <typename T>
static int dispatch_vec(const MaskedParams& p, cudaStream_t st, const char* what) {
  constexpr int VW = sizeof(T) == 4 ? 4 : 8;
  const bool vec = p.D % VW == 0 &&
                   ((reinterpret_cast<uintptr_t>(p.kp) | reinterpret_cast<uintptr_t>(p.vp)) & 15) == 0;
  if (p.unit_tokens * p.G > kVecMost) return vec ? dispatch_tile<T, true>(p, st, what) : dispatch_tile<T, false>(p, st, what);
  if (!vec) return launch_vec<T, 1, 32, 8>(p, st, what);
  // eight lanes a key where registers allow (three shuffles a score, four keys at a time)
  const int n = p.D / VW;
  if (n <= 8) return launch_vec<T, VW, 8, 1>(p, st, what);
  if constexpr (sizeof(T) == 4) {
    if (n <= 16) return launch_vec<T, VW, 8, 2>(p, st, what);
    if (n <= 32) return launch_vec<T, VW, 16, 2>(p, st, what);
    return launch_vec<T, VW, 32, 2>(p, st, what);
  }
  if (n <= 16) return launch_vec<T, VW, 16, 1>(p, st, what);
  if (n <= 32) return launch_vec<T, VW, 32, 1>(p, st, what);
  return fail(NF_EUNSUPPORTED, "%s: head_dim %d > 256", what, p.D);
}

constexpr int kMaskedMaxHeads = 1 << 12;

static int masked_check(const NfMaskedArgs* a, bool tree, const char* what, MaskedParams& p) {
  if (!a) return fail(NF_EINVAL, "%s: null argument struct", what);
  const size_t es = dtype_size(a->dtype);
  if (!es) return fail(NF_EINVAL, "%s: bad dtype %d", what, a->dtype);
  if (a->num_q_heads <= 0 || a->num_kv_heads <= 0 || a->num_q_heads % a->num_kv_heads ||
      a->num_q_heads > kMaskedMaxHeads)
    return fail(NF_EINVAL, "%s: num_q_heads (%d) must be a positive multiple of num_kv_heads (%d), at most %d", what,
                a->num_q_heads, a->num_kv_heads, kMaskedMaxHeads);
  if (a->head_dim <= 0 || a->head_dim > 256)
    return fail(NF_EUNSUPPORTED, "%s: head_dim %d (1 to 256)", what, a->head_dim);
  if (a->block_size <= 0 || a->num_blocks <= 0 || a->max_blocks_per_seq <= 0 || a->num_slots <= 0 || a->num_rows <= 0)
    return fail(NF_EINVAL, "%s: sizes must be positive", what);
  if (a->max_units < 0 || a->max_items < 0 || a->max_merge < 0 || a->ws_rows < 0 ||
      a->max_units + (int64_t)a->max_items <= 0)
    return fail(NF_EINVAL, "%s: work list sizes must not be negative, and not all zero", what);
  if (a->max_units && (a->unit_tokens <= 0 || (int64_t)a->unit_tokens * a->num_q_heads > (1 << 20)))
    return fail(NF_EINVAL, "%s: unit_tokens (%d) must be positive, and at most 2^20 / num_q_heads", what, a->unit_tokens);
  if (!a->out || !a->q || !a->k_pool || !a->v_pool || !a->block_tables || !a->counts || !a->queue ||
      !a->status || (a->max_units && (!a->units || !a->unit_shares)) ||
      (a->max_items && (!a->items || !a->item_shares)) || (a->max_merge && !a->merge) ||
      (a->ws_rows && !a->ws))
    return fail(NF_EINVAL, "%s: null pointer argument", what);
  if (a->q_row_stride < 0 || a->out_row_stride < 0) return fail(NF_EINVAL, "%s: negative row stride", what);
  if (!isfinite(a->scale)) return fail(NF_EINVAL, "%s: scale is not finite", what);
  if (tree && (!a->masks || a->mask_words <= 0)) return fail(NF_EINVAL, "%s: null mask words", what);
  if (!tree && (a->window <= 0 || a->sinks < 0))
    return fail(NF_EINVAL, "%s: window (%d) must be positive and sinks (%d) not negative", what, a->window, a->sinks);
  auto al = [](const void* ptr, size_t n) { return (reinterpret_cast<uintptr_t>(ptr) % n) == 0; };
  if (!al(a->units, 16) || !al(a->items, 16) || !al(a->merge, 16) || !al(a->ws, 16) ||
      !al(a->masks, 4) || !al(a->counts, 4) ||
      !al(a->unit_shares, 4) || !al(a->item_shares, 4))
    return fail(NF_EINVAL, "%s: work lists and workspace must be 16-byte aligned", what);
  if (!al(a->q, es) || !al(a->out, es) || !al(a->k_pool, es) || !al(a->v_pool, es))
    return fail(NF_EINVAL, "%s: tensors must be aligned to their elements", what);
  p = MaskedParams{};
  p.out = static_cast<char*>(a->out);
  p.out_stride = a->out_row_stride;
  p.q = static_cast<const char*>(a->q);
  p.q_stride = a->q_row_stride;
  p.kp = static_cast<const char*>(a->k_pool);
  p.vp = static_cast<const char*>(a->v_pool);
  p.rows = a->num_rows;
  p.Hq = a->num_q_heads;
  p.Hkv = a->num_kv_heads;
  p.D = a->head_dim;
  p.G = p.Hq / p.Hkv;
  p.bs = a->block_size;
  p.num_blocks = a->num_blocks;
  p.bt = a->block_tables;
  p.num_slots = a->num_slots;
  p.max_blocks = a->max_blocks_per_seq;
  p.units = a->units;
  p.max_units = a->max_units;
  p.unit_tokens = a->unit_tokens;
  p.items = a->items;
  p.max_items = a->max_items;
  p.merge = a->merge;
  p.max_merge = a->max_merge;
  p.unit_shares = a->unit_shares;
  p.item_shares = a->item_shares;
  p.counts = a->counts;
  p.masks = a->masks;
  p.mask_words = tree ? a->mask_words : 0;
  p.tree = tree;
  // positions stay below 2^30, so windows and sinks beyond it mean the same and no sum of them overflows
  p.window = a->window < (1 << 30) ? a->window : 1 << 30;
  p.sinks = a->sinks < (1 << 30) ? a->sinks : 1 << 30;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.ws = a->ws;
  p.ws_rows = a->ws_rows;
  p.DP = (a->head_dim + 3) / 4 * 4 + 4;
  p.queue = a->queue;
  p.status = a->status;
  return NF_OK;
}

static int masked_attention(const NfMaskedArgs* a, bool tree, const char* what, void* stream) {
  MaskedParams p;
  int rc = masked_check(a, tree, what, p);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.max_items) {
    rc = launch_masked_tc(p, a->dtype, stream, what);
    if (rc) return rc;
  }
  if (p.max_units) {
    rc = launch_masked_tma(p, a->dtype, stream, what);
    if (rc == NF_EUNSUPPORTED) switch (a->dtype) {
      case NF_F32: rc = dispatch_vec<float>(p, st, what); break;
      case NF_F16: rc = dispatch_vec<__half>(p, st, what); break;
      default: rc = dispatch_vec<__nv_bfloat16>(p, st, what); break;
    }
    if (rc) return rc;
  }
  if (p.max_merge) {
    switch (a->dtype) {
      case NF_F32: return launch_merge<float>(p, a->max_parts, st, what);
      case NF_F16: return launch_merge<__half>(p, a->max_parts, st, what);
      default: return launch_merge<__nv_bfloat16>(p, a->max_parts, st, what);
    }
  }
  return ok();
}

}  // namespace nf

extern "C" int nf_masked_limits(int32_t dtype, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                int32_t block_size, int32_t* unit_rows, int32_t* item_rows) {
  using namespace nf;
  if (!unit_rows || !item_rows) return fail(NF_EINVAL, "nf_masked_limits: null pointer argument");
  if (!dtype_size(dtype)) return fail(NF_EINVAL, "nf_masked_limits: bad dtype %d", dtype);
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || num_q_heads > kMaskedMaxHeads)
    return fail(NF_EINVAL, "nf_masked_limits: num_q_heads (%d) must be a positive multiple of num_kv_heads (%d), at most %d",
                num_q_heads, num_kv_heads, kMaskedMaxHeads);
  if (head_dim <= 0 || head_dim > 256) return fail(NF_EUNSUPPORTED, "nf_masked_limits: head_dim %d (1 to 256)", head_dim);
  if (block_size <= 0) return fail(NF_EINVAL, "nf_masked_limits: block_size must be positive");
  const int G = num_q_heads / num_kv_heads;
  *unit_rows = masked_tma_rows(dtype, num_q_heads, num_kv_heads, head_dim, block_size);
  if (!*unit_rows) *unit_rows = G > kVecRows ? G : kVecRows;
  *item_rows = masked_tc_rows(dtype, num_q_heads, num_kv_heads, head_dim, block_size);
  return ok();
}

extern "C" int nf_window_attention(const NfMaskedArgs* args, void* stream) {
  return nf::masked_attention(args, false, "nf_window_attention", stream);
}

extern "C" int nf_tree_attention(const NfMaskedArgs* args, void* stream) {
  return nf::masked_attention(args, true, "nf_tree_attention", stream);
}
