// Pieces shared by the operators that bound a sequence's cache (windowed
// attention, attention weights, eviction): which keys a row sees, and the
// checks of values that lie in device memory.
#pragma once

#include "ms_attention_common.cuh"

namespace ms {

// Pages that hold a key which positions [first_pos, end) see, under "j <= p and
// (p - j < window or j < sinks)": sink pages [0, sink_pages), then pages
// [first_page, ...) to the end.  Where the two meet, everything from page 0 on
// is one run (sink_pages = 0).  Virtual page i of a row (tile) is
// page_at(i); virtual key v = 16 i + slot.
struct VisiblePages {
  int sink_pages = 0;
  int first_page = 0;
  int count = 0;
  VisiblePages() = default;
  __device__ __forceinline__ VisiblePages(int first_pos, int end, int window, int sinks) {
    const int low = lowest_key(first_pos, window);
    first_page = low / attn::kBS;
    sink_pages = (min(sinks, low) + attn::kBS - 1) / attn::kBS;
    if (sink_pages >= first_page) sink_pages = first_page = 0;
    count = sink_pages + (end + attn::kBS - 1) / attn::kBS - first_page;
  }
  // first key of the window of the row at position pos
  static __device__ __forceinline__ int lowest_key(int pos, int window) {
    return window > 0 ? max(0, pos + 1 - window) : 0;
  }
  __device__ __forceinline__ int page_at(int i) const { return i < sink_pages ? i : i - sink_pages + first_page; }
  // what to add to the key of a page behind the sinks to get its virtual key
  __device__ __forceinline__ int shift() const { return (sink_pages - first_page) * attn::kBS; }
};

// Rows of one call that name the same table row: the first one counts.  Every
// thread of the CTA calls this; true when an earlier row that holds anything
// (a padded batch's rows do not) names `table_row`.
__device__ __forceinline__ bool table_row_repeated(const int32_t *row_table, const int32_t *row_ctx, int row,
                                                   int table_row) {
  int found = 0;
  if (row_table)
    for (int i = threadIdx.x; i < row; i += blockDim.x) found |= row_table[i] == table_row && row_ctx[i] > 0;
  return __syncthreads_or(found) != 0;
}

// bits 0 .. n - 1 set (none for n <= 0, all from n = 32 on)
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : 0xffffffffu >> (32 - min(n, 32)); }

// ---- thread-block clusters ------------------------------------------------------
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
// the 32-bit value at `p` (this CTA's shared memory) in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t peer_u32(const uint32_t *p, int rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(attn::smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint4 peer_u4(const uint32_t *p, int rank) {
  uint32_t a;
  uint4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(attn::smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ float peer_f32(const float *p, int rank) {
  return __uint_as_float(peer_u32(reinterpret_cast<const uint32_t *>(p), rank));
}

inline bool head_layout_ok(int num_heads, int num_kv_heads, int head_dim, int block_size, int dtype) {
  if (num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 || block_size != attn::kBS) return false;
  const int g = num_heads / num_kv_heads;
  if (g != 1 && g != 2 && g != 4 && g != 7 && g != 8) return false;
  if (head_dim != 64 && head_dim != 128) return false;
  return dtype == MS_DTYPE_F32 || dtype == MS_DTYPE_BF16 || dtype == MS_DTYPE_F16;
}
inline bool ptr16(const void *p) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// 32-bit elements, as of tables, contexts, weights and positions
inline bool ptr4(const void *p) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % 4 == 0; }
// pools and block tables of one call; 32-bit page x head tiles, as the TMA coordinates hold them
inline bool pools_ok(const void *k_pool, const void *v_pool, int64_t pool_blocks, int num_kv_heads,
                     const int32_t *block_tables, int table_rows, int max_blocks_per_seq) {
  return ptr16(k_pool) && ptr16(v_pool) && ptr4(block_tables) && pool_blocks > 0 && table_rows > 0 &&
         max_blocks_per_seq > 0 && max_blocks_per_seq <= (1 << 26) && num_kv_heads > 0 &&
         pool_blocks <= ((int64_t(1) << 31) - 1) / num_kv_heads;
}

namespace attn {
// windowed build of the tcgen05 prefill kernel (ms_prefill_tc5.cu); arguments checked, status set
cudaError_t launch_window_prefill_tc5(const WindowArgs &a, cudaStream_t stream);
}  // namespace attn

}  // namespace ms
