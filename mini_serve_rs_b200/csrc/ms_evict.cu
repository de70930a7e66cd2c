// K7: eviction from the paged cache by accumulated attention weight.
//
// Per (sequence, kv head), with n slots of which `keep` stay: rank the slots
// by (protected, weight, lowest slot first) and keep the best.  A kept slot
// below keep stays where it is; the kept slots from keep on ("movers") go, in
// order, into the evicted slots below keep ("holes"), in order.  There are as
// many of one as of the other, a mover's source is never a hole and a hole is
// never a source, so the copies are independent of one another and only what
// has to move moves; attention does not depend on the order of its keys.
//
// One CTA per (sequence, kv head).  The rank of a slot is a 32-bit key whose
// unsigned order is the order of the weights (protected slots: the largest
// key).  The keep-th largest key T is found bit by bit: 32 counts of the keys
// >= a candidate, held in shared memory.  Slots above T stay, and of the slots
// equal to T the lowest ones that still fit.
#include "ms_window.cuh"

namespace ms {
namespace {

constexpr int kThreads = 1024;
constexpr int kMaxSlots = 49152;  // keys of one CTA in shared memory

struct EvictParams {
  unsigned char *k_pool, *v_pool;
  int64_t pool_blocks;
  const int32_t *block_tables;
  int table_rows, max_blocks_per_seq;
  const int32_t *row_table, *row_ctx, *row_next, *row_known;
  int num_rows, max_ctx, keep, sinks, recent;
  const float *w_in;
  float *w_out;
  const int32_t *pos_in;
  int32_t *pos_out;
  int64_t stride;
  int num_kv_heads;
  int row_bytes;  // head_dim * element size
  int32_t *lists;  // [rows][kv heads][2][max_ctx]: holes, movers
  unsigned *status;
};

// unsigned order of the result = order of the weights; -0 as 0, every NaN above infinity
__device__ __forceinline__ uint32_t rank_key(float w) {
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int block_count(int v, int *part) {
  v = __reduce_add_sync(kFull, v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int t = __reduce_add_sync(kFull, part[threadIdx.x & 31]);
  __syncthreads();
  return t;
}

// number of set flags in the threads before this one; total over the CTA in `total`
__device__ __forceinline__ int block_rank(bool flag, int *part, int &total) {
  const unsigned b = __ballot_sync(kFull, flag);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) part[warp] = __popc(b);
  __syncthreads();
  const int c = part[lane];
  const int before = __reduce_add_sync(kFull, lane < warp ? c : 0);
  total = __reduce_add_sync(kFull, c);
  __syncthreads();
  return before + __popc(b & ((1u << lane) - 1));
}

__global__ void __launch_bounds__(kThreads) evict_kernel(EvictParams p) {
  extern __shared__ uint32_t keys[];
  __shared__ int part[32];
  const int row = blockIdx.x, h = blockIdx.y, t = threadIdx.x;
  const int n = p.row_ctx[row], next = p.row_next[row], trow = p.row_table ? p.row_table[row] : row;
  const int known = p.row_known ? p.row_known[row] : 0;
  bool ok = n >= 0 && n <= p.max_ctx && trow >= 0 && trow < p.table_rows && known >= 0 && next >= n;
  if (table_row_repeated(p.row_table, row, trow)) ok = false;
  if (!ok) {
    if (t == 0) atomicOr(p.status, kStatusBadIndex);
    return;
  }
  const size_t base = (size_t(trow) * p.num_kv_heads + h) * size_t(p.stride);
  const float *w_in = p.w_in + base;
  float *w_out = p.w_out + base;
  const int32_t *pos_in = p.pos_in ? p.pos_in + base : nullptr;
  int32_t *pos_out = p.pos_out + base;
  auto position = [&](int j) { return j < known ? pos_in[j] : next - n + j; };
  if (n <= p.keep) {  // nothing to evict
    for (int j = t; j < n; j += kThreads) {
      w_out[j] = w_in[j];
      pos_out[j] = position(j);
    }
    return;
  }
  for (int j = t; j < n; j += kThreads) {
    const int pos = position(j);
    keys[j] = pos < p.sinks || pos >= next - p.recent ? 0xffffffffu : rank_key(w_in[j]);
  }
  __syncthreads();
  // T = the largest value that at least keep keys reach
  uint32_t T = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = T | (1u << bit);
    int v = 0;
    for (int j = t; j < n; j += kThreads) v += keys[j] >= c;
    if (block_count(v, part) >= p.keep) T = c;
  }
  int above = 0;
  for (int j = t; j < n; j += kThreads) above += keys[j] > T;
  const int ties = p.keep - block_count(above, part);  // slots equal to T that stay

  int32_t *holes = p.lists + (size_t(row) * p.num_kv_heads + h) * 2 * size_t(p.max_ctx), *movers = holes + p.max_ctx;
  int seen = 0, nh = 0, nm = 0;  // equal slots, holes, movers so far
  for (int j0 = 0; j0 < n; j0 += kThreads) {
    const int j = j0 + t;
    const uint32_t key = j < n ? keys[j] : 0;
    int total;
    const int tie = seen + block_rank(j < n && key == T, part, total);
    seen += total;
    const bool kept = j < n && (key > T || (key == T && tie < ties));
    const bool hole = j < p.keep && !kept, mover = j >= p.keep && kept;
    const int ih = nh + block_rank(hole, part, total);
    nh += total;
    if (hole) holes[ih] = j;
    const int im = nm + block_rank(mover, part, total);
    nm += total;
    if (mover) movers[im] = j;
    if (j < p.keep && kept) {
      w_out[j] = w_in[j];
      pos_out[j] = position(j);
    }
  }
  __syncthreads();
  const int32_t *table = p.block_tables + size_t(trow) * p.max_blocks_per_seq;
  const int chunks = p.row_bytes / 16;
  for (int i = t; i < nm; i += kThreads) {
    const int to = holes[i], from = movers[i];
    w_out[to] = w_in[from];
    pos_out[to] = position(from);
  }
  for (int i = t; i < nm * chunks; i += kThreads) {
    const int to = holes[i / chunks], from = movers[i / chunks], c = i % chunks;
    const int pt = table[to / attn::kBS], pf = table[from / attn::kBS];
    if (pt < 0 || pt >= p.pool_blocks || pf < 0 || pf >= p.pool_blocks) {
      atomicOr(p.status, kStatusBadIndex);
      continue;
    }
    const size_t dst = ((size_t(pt) * p.num_kv_heads + h) * attn::kBS + to % attn::kBS) * p.row_bytes + 16 * c;
    const size_t src = ((size_t(pf) * p.num_kv_heads + h) * attn::kBS + from % attn::kBS) * p.row_bytes + 16 * c;
    *reinterpret_cast<uint4 *>(p.k_pool + dst) = *reinterpret_cast<const uint4 *>(p.k_pool + src);
    *reinterpret_cast<uint4 *>(p.v_pool + dst) = *reinterpret_cast<const uint4 *>(p.v_pool + src);
  }
  __syncthreads();  // weights of the movers are read: weight_out may be weight_in
  for (int j = p.keep + t; j < n; j += kThreads) w_out[j] = 0.f;
}

}  // namespace

int64_t evict_workspace_bytes(int num_rows, int num_kv_heads, int max_ctx) {
  if (num_rows <= 0 || num_kv_heads <= 0 || max_ctx <= 0) return 0;
  return int64_t(num_rows) * num_kv_heads * 2 * max_ctx * int64_t(sizeof(int32_t));
}

}  // namespace ms

extern "C" int64_t ms_evict_workspace_bytes(int32_t num_rows, int32_t num_kv_heads, int32_t max_ctx) {
  return ms::evict_workspace_bytes(num_rows, num_kv_heads, max_ctx);
}

extern "C" int ms_launch_evict(void *k_pool, void *v_pool, int64_t pool_blocks, const int32_t *block_tables,
                               int32_t table_rows, int32_t max_blocks_per_seq, const int32_t *row_table,
                               const int32_t *row_ctx, const int32_t *row_next, const int32_t *row_known,
                               int32_t num_rows, int32_t max_ctx, int32_t keep, int32_t sinks, int32_t recent,
                               const float *weight_in, float *weight_out, const int32_t *pos_in, int32_t *pos_out,
                               int64_t stride, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                               void *workspace, int64_t workspace_bytes, int32_t dtype, void *stream) {
  using namespace ms;
  if (num_rows < 0 || max_ctx < 0) return int(cudaErrorInvalidValue);
  if (num_rows == 0 || max_ctx == 0) return 0;
  if (!head_layout_ok(num_kv_heads, num_kv_heads, head_dim, block_size, dtype) || num_kv_heads > 65535 ||
      !pools_ok(k_pool, v_pool, pool_blocks, num_kv_heads, block_tables, table_rows, max_blocks_per_seq) ||
      max_ctx > kMaxSlots || max_ctx > int64_t(max_blocks_per_seq) * attn::kBS || stride < max_ctx ||
      (!row_table && table_rows < num_rows) || !row_ctx || !row_next || (row_known && !pos_in) || !weight_in ||
      !weight_out || !pos_out || keep <= 0 || sinks < 0 || recent < 0 || int64_t(sinks) + recent > keep ||
      workspace == nullptr || workspace_bytes < evict_workspace_bytes(num_rows, num_kv_heads, max_ctx))
    return int(cudaErrorInvalidValue);
  EvictParams p{};
  p.k_pool = static_cast<unsigned char *>(k_pool);
  p.v_pool = static_cast<unsigned char *>(v_pool);
  p.pool_blocks = pool_blocks;
  p.block_tables = block_tables;
  p.table_rows = table_rows;
  p.max_blocks_per_seq = max_blocks_per_seq;
  p.row_table = row_table;
  p.row_ctx = row_ctx;
  p.row_next = row_next;
  p.row_known = row_known;
  p.num_rows = num_rows;
  p.max_ctx = max_ctx;
  p.keep = keep;
  p.sinks = sinks;
  p.recent = recent;
  p.w_in = weight_in;
  p.w_out = weight_out;
  p.pos_in = pos_in;
  p.pos_out = pos_out;
  p.stride = stride;
  p.num_kv_heads = num_kv_heads;
  p.row_bytes = head_dim * (dtype == MS_DTYPE_F32 ? 4 : 2);
  p.lists = static_cast<int32_t *>(workspace);
  cudaError_t e = standalone_status_word(&p.status);
  if (e != cudaSuccess) return int(e);
  const size_t smem = size_t(max_ctx) * sizeof(uint32_t);
  e = cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSlots * 4);
  if (e != cudaSuccess) return int(e);
  evict_kernel<<<dim3(num_rows, num_kv_heads), kThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  return int(cudaGetLastError());
}
