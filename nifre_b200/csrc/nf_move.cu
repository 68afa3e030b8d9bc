// Copies of cache rows within the block pools, all layers and both pools in
// one launch (nf_kv_move): block copies, forks of partly filled blocks,
// accepted paths of drafted tokens moved together, pool compaction.
//
// Bound by HBM: each byte is read once and written once.  A CTA takes tiles
// of kTileCols 16-byte columns of a record's rows, every thread with four
// loads in flight before its stores; a CTA a tile (1000 blocks of 16 layers, 1.05
// GB: 161 us, the measured copy bandwidth; a grid of eight CTAs an SM that walk
// the tiles 183 us, cache hints and eight loads no better).  Records that continue a run are ordered
// after the ones before them: the CTA that holds the run's tile walks its
// records row by row, each thread on its own column, so rows may move onto
// rows that the run has read already (no other thread touches the column).
// Short lists travel as kernel arguments: a fork of a few sequences then
// costs one launch and no upload.
#include "nf_common.cuh"
#include "nf_internal.h"

namespace nf {

constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 4;
constexpr int kTileCols = kMoveThreads * kMoveUnroll;
constexpr int kListMoves = NF_MOVE_LIST;  // records that fit the kernel arguments
constexpr int kListPos = NF_MOVE_LIST;

struct MoveParams {
  char* kp;
  char* vp;
  long long layer_stride;
  int layers;
  long long row_bytes, pool_rows;
  int n_moves, max_rows;
  int n_tiles;  // column tiles of the longest record
  int n_pos;
  long long* pos_out;
  int num_slots;
  int* status;
};

struct MoveLists {  // in device memory
  const int4* moves;
  const int2* pos;
  __device__ __forceinline__ int4 move(int i) const { return __ldg(moves + i); }
  __device__ __forceinline__ int2 at(int i) const { return __ldg(pos + i); }
};
struct MoveArgs {  // in the kernel's arguments
  int4 moves[kListMoves];
  int2 pos[kListPos];
  __device__ __forceinline__ int4 move(int i) const { return moves[i]; }
  __device__ __forceinline__ int2 at(int i) const { return pos[i]; }
};

struct BlockIds {  // block copies: source and destination ids in device memory
  const int* src;
  const int* dst;
  __device__ __forceinline__ int4 move(int i) const { return make_int4(__ldg(src + i), __ldg(dst + i), 1, 0); }
  __device__ __forceinline__ int2 at(int) const { return make_int2(-1, 0); }
};

__device__ __forceinline__ bool move_ok(const MoveParams& p, const int4& m) {
  return m.z >= 0 && m.z <= p.max_rows && m.x >= 0 && m.y >= 0 && m.x <= p.pool_rows - m.z && m.y <= p.pool_rows - m.z;
}

// V: a column's type (16 bytes where rows and pools allow it, else 2).
template <typename V, typename L>
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const __grid_constant__ MoveParams p,
                                                               const __grid_constant__ L lists) {
  pdl_launch_dependents();
  pdl_wait();  // the rows may come from the launch before this one
  const long long cols = p.row_bytes / (long long)sizeof(V);
  const long long total = (long long)p.n_moves * p.layers * 2 * p.n_tiles;
  for (long long tile = blockIdx.x; tile < total; tile += gridDim.x) {
    const int x = (int)(tile % p.n_tiles);
    const long long r = tile / p.n_tiles;
    const int side = (int)(r & 1), layer = (int)((r >> 1) % p.layers), i0 = (int)((r >> 1) / p.layers);
    const int4 mv = lists.move(i0);
    if (mv.w) continue;  // a later record of a run
    V* pool = reinterpret_cast<V*>((side ? p.vp : p.kp) + layer * p.layer_stride);
    const long long c0 = (long long)x * kTileCols + threadIdx.x;
    const bool run = !std::is_same<L, BlockIds>::value && i0 + 1 < p.n_moves && lists.move(i0 + 1).w != 0;
    if (!run && !move_ok(p, mv)) {
      if (threadIdx.x == 0 && x == 0)
        atomicOr(p.status, std::is_same<L, BlockIds>::value ? NF_STATUS_BAD_BLOCK : NF_STATUS_BAD_SLOT);
      continue;
    }
    if (!run && abs(mv.y - mv.x) >= mv.z) {  // one record, source and destination apart
      const long long n = mv.z * cols;
      const V* src = pool + mv.x * cols;
      V* dst = pool + mv.y * cols;
      V v[kMoveUnroll];
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u)
        if (c0 + u * kMoveThreads < n) v[u] = src[c0 + u * kMoveThreads];
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u)
        if (c0 + u * kMoveThreads < n) dst[c0 + u * kMoveThreads] = v[u];
      continue;
    }
    // a run: its rows in order, a column a thread (tiles past one row's columns have nothing to do)
    for (int i = i0; i < p.n_moves; ++i) {
      const int4 m = i == i0 ? mv : lists.move(i);
      if (i > i0 && !m.w) break;
      if (!move_ok(p, m)) {
        if (threadIdx.x == 0 && x == 0) atomicOr(p.status, NF_STATUS_BAD_SLOT);
        continue;
      }
      for (int row = 0; row < m.z; ++row)
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
          const long long c = c0 + u * kMoveThreads;
          if (c < cols) pool[(m.y + row) * cols + c] = pool[(m.x + row) * cols + c];
        }
    }
  }
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.n_pos; i += kMoveThreads) {
      const int2 v = lists.at(i);
      if (v.x < 0 || v.x >= p.num_slots)
        atomicOr(p.status, NF_STATUS_BAD_SLOT);
      else
        p.pos_out[v.x] = v.y;
    }
}

template <typename V, typename L>
static int launch_move(const MoveParams& p, const L& lists, cudaStream_t st) {
  long long blocks = (long long)p.n_moves * p.layers * 2 * p.n_tiles;
  if (blocks > (1 << 30)) blocks = 1 << 30;
  if (blocks < 1) blocks = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kv_move_kernel<V, L>, p, lists);
  if (e != cudaSuccess) return fail(NF_ECUDA, "nf_kv_move: launch: %s", cudaGetErrorString(e));
  return check_launch("nf_kv_move");
}

static int fill_move(MoveParams& p, bool& wide, void* k_pool, void* v_pool, int64_t layer_stride, int num_layers,
                     int64_t row_bytes, int64_t pool_rows, int n_moves, int max_rows, int* status) {
  auto al = [](const void* ptr, size_t n) { return (reinterpret_cast<uintptr_t>(ptr) % n) == 0; };
  if (!k_pool || !v_pool || !status) return fail(NF_EINVAL, "nf_kv_move: null pointer argument");
  if (num_layers <= 0 || row_bytes <= 0 || row_bytes % 2 || row_bytes > (1ll << 40) || pool_rows <= 0 ||
      pool_rows > INT32_MAX || layer_stride < 0)
    return fail(NF_EINVAL, "nf_kv_move: sizes must be positive, and rows of an even number of bytes");
  if (!al(k_pool, 2) || !al(v_pool, 2) || layer_stride % 2)
    return fail(NF_EINVAL, "nf_kv_move: pools must be 2-byte aligned");
  wide = row_bytes % 16 == 0 && layer_stride % 16 == 0 && al(k_pool, 16) && al(v_pool, 16);
  p = MoveParams{};
  p.kp = static_cast<char*>(k_pool);
  p.vp = static_cast<char*>(v_pool);
  p.layer_stride = layer_stride;
  p.layers = num_layers;
  p.row_bytes = row_bytes;
  p.pool_rows = pool_rows;
  p.n_moves = n_moves;
  p.max_rows = max_rows;
  const long long most = (max_rows < pool_rows ? max_rows : pool_rows) * (row_bytes / (wide ? 16 : 2));
  const long long tiles = (most + kTileCols - 1) / kTileCols;
  if (tiles > INT32_MAX) return fail(NF_EINVAL, "nf_kv_move: records of too many bytes");
  p.n_tiles = tiles < 1 ? 1 : (int)tiles;
  p.status = status;
  return NF_OK;
}

}  // namespace nf

extern "C" int nf_copy_blocks(void* k_pool, void* v_pool, int64_t layer_stride, int32_t num_layers,
                              int64_t block_bytes, int32_t num_blocks, const int32_t* src, const int32_t* dst,
                              int32_t n, int32_t* status, void* stream) {
  using namespace nf;
  if (n < 0 || (n && (!src || !dst))) return fail(NF_EINVAL, "nf_copy_blocks: null or negative list");
  MoveParams p;
  bool wide;
  const int rc = fill_move(p, wide, k_pool, v_pool, layer_stride, num_layers, block_bytes, num_blocks, n, 1, status);
  if (rc) return rc;
  if (n == 0) return ok();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const BlockIds l{src, dst};
  return wide ? launch_move<uint4>(p, l, st) : launch_move<unsigned short>(p, l, st);
}

extern "C" int nf_kv_move(void* k_pool, void* v_pool, int64_t layer_stride, int32_t num_layers, int64_t row_bytes,
                          int64_t pool_rows, const int32_t* moves, int32_t n_moves, int32_t max_rows,
                          const int32_t* pos, int32_t n_pos, int64_t* pos_out, int32_t num_slots, int32_t on_device,
                          int32_t* status, void* stream) {
  using namespace nf;
  if (n_moves < 0 || n_pos < 0 || max_rows < 0) return fail(NF_EINVAL, "nf_kv_move: negative count");
  if ((n_moves && !moves) || (n_pos && (!pos || !pos_out || num_slots <= 0)))
    return fail(NF_EINVAL, "nf_kv_move: null list");
  if (!on_device && (n_moves > kListMoves || n_pos > kListPos))
    return fail(NF_EINVAL, "nf_kv_move: lists of %d and %d records: more than %d go in device memory", n_moves, n_pos,
                kListMoves);
  if (n_moves == 0 && n_pos == 0) return ok();
  auto al = [](const void* ptr, size_t n) { return (reinterpret_cast<uintptr_t>(ptr) % n) == 0; };
  if (on_device && (!al(moves, 16) || !al(pos, 8)))
    return fail(NF_EINVAL, "nf_kv_move: lists in device memory must be 16- and 8-byte aligned");
  MoveParams p;
  bool wide;
  const int rc = fill_move(p, wide, k_pool, v_pool, layer_stride, num_layers, row_bytes, pool_rows, n_moves, max_rows, status);
  if (rc) return rc;
  p.n_pos = n_pos;
  p.pos_out = reinterpret_cast<long long*>(pos_out);
  p.num_slots = num_slots;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (on_device) {
    const MoveLists l{reinterpret_cast<const int4*>(moves), reinterpret_cast<const int2*>(pos)};
    return wide ? launch_move<uint4>(p, l, st) : launch_move<unsigned short>(p, l, st);
  }
  MoveArgs l;
  for (int i = 0; i < n_moves; ++i) {
    const int32_t* m = moves + 4 * i;
    if (m[2] > max_rows) return fail(NF_EINVAL, "nf_kv_move: a record of %d rows (max_rows %d)", m[2], max_rows);
    l.moves[i] = make_int4(m[0], m[1], m[2], m[3]);
  }
  for (int i = 0; i < n_pos; ++i) l.pos[i] = make_int2(pos[2 * i], pos[2 * i + 1]);
  return wide ? launch_move<uint4>(p, l, st) : launch_move<unsigned short>(p, l, st);
}
