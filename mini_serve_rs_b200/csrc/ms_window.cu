// K3w / K3pw / K3a: attention over a bounded part of the paged cache.
//
//   o = sum_j softmax_j(scale q . k_j) v_j   over  j <= p, p - j < window or j < sinks
//
// for single tokens (K3w) and for the tiles of prompt chunks (K3pw), and over
// the whole cache with W[j] += sum over the kv head's query heads of key j's
// softmax weight (K3a).
//
// K3pw is the windowed build of the tcgen05 prefill kernel
// (ms_prefill_tc5.cu); this file checks its arguments.  Single tokens:
// one CTA per (row, kv head); its warps take the visible keys in turn, a lane
// holding head_dim / 32 dims, every query head of the kv head served by one
// read of K and V.  Softmax is online in base 2; the warps merge in shared
// memory.  K3a keeps the raw scores in the workspace and turns them into
// weights once the row's maximum and sum are known.
#include "ms_window.cuh"

namespace ms {
namespace {

constexpr int kMaxGroup = 8;

struct RowsParams {
  WindowArgs a;
  int group;
  float qscale;
  unsigned *status;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) window_rows_kernel(RowsParams p) {
  constexpr int DPL = D / 32, W = 4;
  const WindowArgs &a = p.a;
  const int kvh = blockIdx.y, G = p.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x, ctx = a.row_ctx[row], trow = a.row_table ? a.row_table[row] : row;
  bool ok = ctx >= 0 && ctx <= a.max_ctx;
  ok = ok && trow >= 0 && trow < a.table_rows;
  if (a.weight_sum && table_row_repeated(a.row_table, row, trow)) ok = false;
  if (!ok) {
    if (threadIdx.x == 0) atomicOr(p.status, kStatusBadIndex);
    return;
  }
  const int32_t *table = a.block_tables + size_t(trow) * a.max_blocks_per_seq;
  const int low = VisiblePages::lowest_key(ctx - 1, a.window);
  const int nsink = min(a.sinks, low), nvis = nsink + ctx - low;
  const T *q = static_cast<const T *>(a.q) + (size_t(row) * a.num_kv_heads + kvh) * G * D;
  T *out = static_cast<T *>(a.out) + (size_t(row) * a.num_kv_heads + kvh) * G * D;
  float *raw = a.weight_sum ? static_cast<float *>(a.workspace) + (size_t(row) * a.num_kv_heads + kvh) * G * a.max_ctx
                            : nullptr;

  float qv[kMaxGroup][DPL], o[kMaxGroup][DPL], m[kMaxGroup], l[kMaxGroup];
#pragma unroll
  for (int g = 0; g < kMaxGroup; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int d = 0; d < DPL; ++d) {
      qv[g][d] = g < G ? Elem<T>::to_f(q[g * D + lane * DPL + d]) : 0.f;
      o[g][d] = 0.f;
    }
  }
  for (int i = warp; i < nvis; i += W) {
    const int key = i < nsink ? i : low + i - nsink;
    const int page = table[key / attn::kBS];
    if (page < 0 || page >= a.pool_blocks) {
      if (lane == 0) atomicOr(p.status, kStatusBadIndex);
      continue;
    }
    const size_t at = ((size_t(page) * a.num_kv_heads + kvh) * attn::kBS + key % attn::kBS) * D + lane * DPL;
    float k[DPL], v[DPL];
#pragma unroll
    for (int d = 0; d < DPL; ++d) {
      k[d] = Elem<T>::to_f(static_cast<const T *>(a.k_pool)[at + d]);
      v[d] = Elem<T>::to_f(static_cast<const T *>(a.v_pool)[at + d]);
    }
#pragma unroll
    for (int g = 0; g < kMaxGroup; ++g) {
      if (g >= G) break;
      float s = 0.f;
#pragma unroll
      for (int d = 0; d < DPL; ++d) s = fmaf(qv[g][d], k[d], s);
      s = warp_sum(s) * p.qscale;
      if (raw && lane == 0) raw[size_t(g) * a.max_ctx + key] = s;
      const float mn = fmaxf(m[g], s), f = exp2f(m[g] - mn), e = exp2f(s - mn);
      l[g] = l[g] * f + e;
      m[g] = mn;
#pragma unroll
      for (int d = 0; d < DPL; ++d) o[g][d] = fmaf(e, v[d], o[g][d] * f);
    }
  }
  __shared__ float so[W][kMaxGroup][D], sm[W][kMaxGroup], sl[W][kMaxGroup];
#pragma unroll
  for (int g = 0; g < kMaxGroup; ++g) {
#pragma unroll
    for (int d = 0; d < DPL; ++d) so[warp][g][lane * DPL + d] = o[g][d];
    if (lane == 0) {
      sm[warp][g] = m[g];
      sl[warp][g] = l[g];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D; i += 128) {
    const int g = i / D, d = i % D;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w][g]);
    for (int w = 0; w < W; ++w) {
      const float f = sm[w][g] == -INFINITY ? 0.f : exp2f(sm[w][g] - M);
      L += f * sl[w][g];
      O += f * so[w][g][d];
    }
    out[i] = Elem<T>::from_f(L > 0.f ? O / L : 0.f);
  }
  if (!raw) return;
  float *sum = a.weight_sum + (size_t(trow) * a.num_kv_heads + kvh) * a.weight_stride;
  for (int key = threadIdx.x; key < ctx; key += 128) {
    const int page = table[key / attn::kBS];
    if (page < 0 || page >= a.pool_blocks) continue;
    float add = 0.f;
    for (int g = 0; g < G; ++g) {
      float M = -INFINITY, L = 0.f;
      for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w][g]);
      for (int w = 0; w < W; ++w) L += sm[w][g] == -INFINITY ? 0.f : exp2f(sm[w][g] - M) * sl[w][g];
      add += exp2f(raw[size_t(g) * a.max_ctx + key] - M) / L;
    }
    sum[key] += add;
  }
}

template <typename T>
cudaError_t launch_rows(const RowsParams &p, cudaStream_t stream) {
  const dim3 grid(p.a.num_rows, p.a.num_kv_heads);
  if (p.a.head_dim == 128) window_rows_kernel<T, 128><<<grid, 128, 0, stream>>>(p);
  else window_rows_kernel<T, 64><<<grid, 128, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_checked(const WindowArgs &a, cudaStream_t stream) {
  RowsParams p{};
  p.a = a;
  p.group = a.num_heads / a.num_kv_heads;
  p.qscale = a.scale * attn::kLog2e;
  p.status = a.status;
  if (!p.status) {
    const cudaError_t e = standalone_status_word(&p.status);
    if (e != cudaSuccess) return e;
  }
  if (a.dtype == MS_DTYPE_F32) return launch_rows<float>(p, stream);
  if (a.dtype == MS_DTYPE_BF16) return launch_rows<__nv_bfloat16>(p, stream);
  return launch_rows<__half>(p, stream);
}

bool common_ok(const WindowArgs &a) {
  return head_layout_ok(a.num_heads, a.num_kv_heads, a.head_dim, a.block_size, a.dtype) && a.num_kv_heads <= 65535 &&
         pools_ok(a.k_pool, a.v_pool, a.pool_blocks, a.num_kv_heads, a.block_tables, a.table_rows,
                  a.max_blocks_per_seq) &&
         ptr16(a.q) && ptr16(a.out) && a.scale > 0.f && a.scale < INFINITY && a.window >= 0 && a.sinks >= 0;
}

}  // namespace

cudaError_t launch_window_attention(const WindowArgs &a, cudaStream_t stream) {
  if (a.num_rows < 0 || a.max_ctx < 0) return cudaErrorInvalidValue;
  if (a.num_rows == 0) return cudaSuccess;
  if (!common_ok(a) || !a.row_ctx || a.tiles || a.max_ctx > int64_t(a.max_blocks_per_seq) * attn::kBS ||
      (!a.row_table && a.table_rows < a.num_rows))
    return cudaErrorInvalidValue;
  if (a.weight_sum && (a.weight_stride < a.max_ctx || !ptr16(a.workspace) ||
                       a.workspace_bytes < attention_weights_workspace_bytes(a.num_rows, a.num_heads, a.max_ctx)))
    return cudaErrorInvalidValue;
  return launch_checked(a, stream);
}

cudaError_t launch_window_prefill(const WindowArgs &args, cudaStream_t stream) {
  WindowArgs a = args;
  if (a.num_tiles < 0) return cudaErrorInvalidValue;
  if (a.num_tiles == 0) return cudaSuccess;
  if (!common_ok(a) || !a.tiles || a.dtype == MS_DTYPE_F32 || a.num_tiles > 65535) return cudaErrorInvalidValue;
  if (!attention_tc_available(a.dtype, a.head_dim, a.num_heads / a.num_kv_heads)) return cudaErrorInvalidValue;
  if (!a.status) {
    const cudaError_t e = standalone_status_word(&a.status);
    if (e != cudaSuccess) return e;
  }
  return attn::launch_window_prefill_tc5(a, stream);
}

int64_t attention_weights_workspace_bytes(int num_rows, int num_heads, int max_ctx) {
  if (num_rows <= 0 || num_heads <= 0 || max_ctx <= 0) return 0;
  const int64_t ctx16 = (int64_t(max_ctx) + 15) / 16 * 16;
  return int64_t(num_rows) * num_heads * ctx16 * int64_t(sizeof(float));
}

}  // namespace ms

// ---------------------------------------------------------------------------
// C ABI
namespace {
ms::WindowArgs pool_args(const void *q, const void *k_pool, const void *v_pool, int64_t pool_blocks,
                         const int32_t *block_tables, int32_t table_rows, int32_t max_blocks_per_seq, void *out,
                         int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size, float scale,
                         int32_t dtype) {
  ms::WindowArgs a{};
  a.q = q;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.pool_blocks = pool_blocks;
  a.block_tables = block_tables;
  a.table_rows = table_rows;
  a.max_blocks_per_seq = max_blocks_per_seq;
  a.out = out;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.scale = scale;
  a.dtype = dtype;
  return a;
}
}  // namespace

extern "C" int ms_launch_window_attention(const void *q, const void *k_pool, const void *v_pool, int64_t pool_blocks,
                                          const int32_t *block_tables, int32_t table_rows, int32_t max_blocks_per_seq,
                                          const int32_t *row_table, const int32_t *row_ctx, int32_t num_rows,
                                          int32_t max_ctx, int32_t window, int32_t sinks, void *out, int32_t num_heads,
                                          int32_t num_kv_heads, int32_t head_dim, int32_t block_size, float scale,
                                          int32_t dtype, void *stream) {
  ms::WindowArgs a = pool_args(q, k_pool, v_pool, pool_blocks, block_tables, table_rows, max_blocks_per_seq, out,
                               num_heads, num_kv_heads, head_dim, block_size, scale, dtype);
  a.row_table = row_table;
  a.row_ctx = row_ctx;
  a.num_rows = num_rows;
  a.max_ctx = max_ctx;
  a.window = window;
  a.sinks = sinks;
  return int(ms::launch_window_attention(a, static_cast<cudaStream_t>(stream)));
}

extern "C" int ms_launch_window_prefill(const void *q, const void *k_pool, const void *v_pool, int64_t pool_blocks,
                                        const int32_t *block_tables, int32_t table_rows, int32_t max_blocks_per_seq,
                                        const int32_t *tiles, int32_t num_tiles, int32_t window, int32_t sinks,
                                        void *out, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                        int32_t block_size, float scale, int32_t dtype, void *stream) {
  ms::WindowArgs a = pool_args(q, k_pool, v_pool, pool_blocks, block_tables, table_rows, max_blocks_per_seq, out,
                               num_heads, num_kv_heads, head_dim, block_size, scale, dtype);
  a.tiles = tiles;
  a.num_tiles = num_tiles;
  a.window = window;
  a.sinks = sinks;
  return int(ms::launch_window_prefill(a, static_cast<cudaStream_t>(stream)));
}

extern "C" int64_t ms_attention_weights_workspace_bytes(int32_t num_rows, int32_t num_heads, int32_t max_ctx) {
  return ms::attention_weights_workspace_bytes(num_rows, num_heads, max_ctx);
}

extern "C" int ms_launch_attention_weights(const void *q, const void *k_pool, const void *v_pool, int64_t pool_blocks,
                                           const int32_t *block_tables, int32_t table_rows,
                                           int32_t max_blocks_per_seq, const int32_t *row_table,
                                           const int32_t *row_ctx, int32_t num_rows, int32_t max_ctx, void *out,
                                           float *weight_sum, int64_t weight_stride, int32_t num_heads,
                                           int32_t num_kv_heads, int32_t head_dim, int32_t block_size, float scale,
                                           void *workspace, int64_t workspace_bytes, int32_t dtype, void *stream) {
  ms::WindowArgs a = pool_args(q, k_pool, v_pool, pool_blocks, block_tables, table_rows, max_blocks_per_seq, out,
                               num_heads, num_kv_heads, head_dim, block_size, scale, dtype);
  a.row_table = row_table;
  a.row_ctx = row_ctx;
  a.num_rows = num_rows;
  a.max_ctx = max_ctx;
  a.weight_sum = weight_sum;
  a.weight_stride = weight_stride;
  a.workspace = workspace;
  a.workspace_bytes = workspace_bytes;
  if (!weight_sum && num_rows != 0) return int(cudaErrorInvalidValue);
  return int(ms::launch_window_attention(a, static_cast<cudaStream_t>(stream)));
}
