// K3w / K3pw / K3a: attention over a bounded part of the paged cache.
//
//   o = sum_j softmax_j(scale q . k_j) v_j   over  j <= p, p - j < window or j < sinks
//
// for single tokens (K3w) and for the tiles of prompt chunks (K3pw), and over
// the whole cache with W[j] += sum over the kv head's query heads of key j's
// softmax weight (K3a).  K3pw is the windowed build of the tcgen05 prefill
// kernel (ms_prefill_tc5.cu); this file checks its arguments.
//
// Single tokens: bound by reading the visible K and V once, so the kernel is
// built around keeping copies in flight.  A cluster of C CTAs serves one (row,
// kv head); CTA c takes the c-th share of the row's visible pages (sink pages,
// then the window's; the others are never touched), its 4 warps take the
// share's pages in turn, each through a private ring of shared-memory stages
// filled by TMA (no multicast) on per-stage mbarriers.  Two stages a warp and
// three CTAs on an SM: 192 KB of copies in flight, and while one CTA joins its
// warps the others stream (three stages and two CTAs: 86 against 79 us on 64
// rows of 28/4 heads behind a 4096-token window, 0.97 of the copy rate).
// One read of K and V serves all query heads of the kv head:
//  * 16-bit: the heads are rows 0..G-1 of an m16 tile, S = Q K^T and O += P V
//    as mma.sync.m16n8k16 on the swizzled tile (16 x 16 x D per page is far
//    below one tcgen05 tile), online softmax in base 2 on the four scores a
//    lane holds;
//  * f32: a lane owns D / 32 dims; partial dot products of 16 tokens are
//    reduced across the warp by a transposed butterfly.  ~2000 cycles a page,
//    so many warps with one 16 KB stage each do better than few with two (24
//    rows, window 1001: 12 warps an SM 29.8 us, 6 warps 35.3).
// The warps merge in shared memory, the CTAs of the cluster read one another's
// maxima, sums and outputs there (distributed shared memory): one launch, no
// workspace, and the split depends on the call's shape only, so equal calls
// give equal bits.
// K3a needs the row's final maximum and sum before a score becomes a weight:
// each CTA writes its raw scores to the workspace and reads them back once the
// cluster has exchanged the maxima and sums.  4 bytes per row, query head and
// key: they stay in L2 for few rows (of 64 rows x 16 heads x 4608 keys, 19 MB,
// 12 MB were written out; 155 us, 0.86 of the copy rate).
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <type_traits>

#include "ms_window.cuh"

namespace ms {
namespace {

using namespace attn;

constexpr int kMaxCluster = 8;
// running maxima start here, not at -infinity: a page whose scores are all -infinity (products below
// the f32 range) then gives 2^-infinity = 0 and no NaN
constexpr float kLowest = -FLT_MAX;

struct RowsParams {
  const void *q, *k_pool, *v_pool;
  const int32_t *block_tables, *row_table, *row_ctx, *row_index;
  void *out;
  float *weight_sum, *raw;  // K3a: accumulators; raw scores [rows][Hkv][G][ctx16]
  int64_t weight_stride;
  unsigned *status;
  int pool_blocks, table_rows, max_blocks_per_seq;
  int max_ctx, ctx16;
  int window, sinks;
  int num_kv_heads, group;
  float qscale;  // softmax scale * log2(e)
  int wait_limit;
};

// ---- one page of one kv head: 16-bit K/V on mma.sync ----------------------------------
template <typename T_, int D_> struct PageTc {
  using T = T_;
  static constexpr int D = D_, WARPS = 4, NSTAGE = D == 128 ? 2 : 3;
  static constexpr int NDH = D / 64, TILE_BYTES = NDH * kHalfBytes, KSTEPS = D / 16, NTD = D / 8;
  // P <= 1 is stored as 2^15 P in f16, whose numbers are of full precision from 2^-14 to 2^16 only
  // (bf16 has f32's range): without it keys 2^-25 as heavy as the heaviest vanished from O but not
  // from the sum.  store() takes the factor out again.
  static constexpr float kScaleP = std::is_same<T, __half>::value ? 32768.f : 1.f;
  uint32_t qa[KSTEPS][2];
  float o[NTD][4];
  float m_run = kLowest, l_run = 0.f;

  __device__ __forceinline__ void init(const T *q, int group, float) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    const T *row = q + (gid < group ? gid : 0) * D;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      qa[kk][0] = gid < group ? *reinterpret_cast<const uint32_t *>(row + kk * 16 + 2 * tig) : 0u;
      qa[kk][1] = gid < group ? *reinterpret_cast<const uint32_t *>(row + kk * 16 + 8 + 2 * tig) : 0u;
    }
#pragma unroll
    for (int nd = 0; nd < NTD; ++nd) o[nd][0] = o[nd][1] = o[nd][2] = o[nd][3] = 0.f;
  }

  static __device__ __forceinline__ void issue(unsigned char *st, const CUtensorMap &kmap, const CUtensorMap &vmap,
                                               const RowsParams &, int page, int kvh, int hkv, uint64_t *bar) {
    mbar_expect_tx(bar, 2 * TILE_BYTES);
#pragma unroll
    for (int dh = 0; dh < NDH; ++dh) {
      tma_load_4d(st + dh * kHalfBytes, &kmap, 0, dh, 0, page * hkv + kvh, bar);
      tma_load_4d(st + TILE_BYTES + dh * kHalfBytes, &vmap, 0, dh, 0, page * hkv + kvh, bar);
    }
  }

  // bits: visible tokens of the page, at least one.  raw: the page's scores of head 0, or null.
  __device__ __forceinline__ void page(unsigned char *st, uint32_t bits, float qscale, float *raw, int raw_stride,
                                       int group) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3, mi = lane >> 3, lr = lane & 7;
    const uint32_t kb = smem_addr(st), vb = kb + TILE_BYTES;
    if (bits != 0xffffu) {
      // what the row does not see may hold anything, NaN included: P = 0 must meet V = 0
      uint4 *vz = reinterpret_cast<uint4 *>(st + TILE_BYTES);
#pragma unroll
      for (int i = lane; i < NDH * kBS * 8; i += 32)
        if (!(bits >> ((i >> 3) & 15) & 1)) vz[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
    }
    // tokens 0..7 and 8..15; even and odd k-steps apart: half the chain of dependent products
    float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    float sd[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int kk = 0; kk < KSTEPS; kk += 2) {
      uint32_t b[4], c[4];
      ldmatrix_x4(b, kb + tile_off((mi >> 1) * 8 + lr, kk * 16 + (mi & 1) * 8));
      ldmatrix_x4(c, kb + tile_off((mi >> 1) * 8 + lr, kk * 16 + 16 + (mi & 1) * 8));
      const uint32_t a[4] = {qa[kk][0], 0u, qa[kk][1], 0u};
      const uint32_t a2[4] = {qa[kk + 1][0], 0u, qa[kk + 1][1], 0u};
      mma_16816<T>(sc[0], a, b[0], b[1]);
      mma_16816<T>(sc[1], a, b[2], b[3]);
      mma_16816<T>(sd[0], a2, c[0], c[1]);
      mma_16816<T>(sd[1], a2, c[2], c[3]);
    }
    // row gid: tokens 2 tig, 2 tig + 1, 8 + 2 tig, 9 + 2 tig
    float sv[4] = {sc[0][0] + sd[0][0], sc[0][1] + sd[0][1], sc[1][0] + sd[1][0], sc[1][1] + sd[1][1]};
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int tk = 2 * tig + (j & 1) + 8 * (j >> 1);
      sv[j] = bits >> tk & 1 ? sv[j] * qscale : -INFINITY;
      mx = fmaxf(mx, sv[j]);
    }
    if (raw && gid < group) {  // (slots past the row's context: inside the 16-slot rounding)
      float *r = raw + size_t(gid) * raw_stride;
      *reinterpret_cast<float2 *>(r + 2 * tig) = make_float2(sv[0], sv[1]);
      *reinterpret_cast<float2 *>(r + 8 + 2 * tig) = make_float2(sv[2], sv[3]);
    }
    mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 2));
    const float m_new = fmaxf(m_run, mx);
    const float alpha = exp2f(m_run - m_new);
    float pj[4], psum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      pj[j] = exp2f(sv[j] - m_new);
      psum += pj[j];
    }
    l_run = l_run * alpha + psum;
    m_run = m_new;
#pragma unroll
    for (int nd = 0; nd < NTD; ++nd) {
      o[nd][0] *= alpha;
      o[nd][1] *= alpha;
    }
    // P is rounded to the K/V type for the tensor cores (the sum above is not): half a step
    // relative per weight, which the result's own rounding matches; in f16 below 2^-29 of the
    // heaviest key half of 2^-39 of that key's weight
    const uint32_t pa[4] = {pack2<T>(pj[0] * kScaleP, pj[1] * kScaleP), 0u, pack2<T>(pj[2] * kScaleP, pj[3] * kScaleP), 0u};
#pragma unroll
    for (int ndp = 0; ndp < NTD / 2; ++ndp) {
      uint32_t b[4];
      ldmatrix_x4_trans(b, vb + tile_off((mi & 1) * 8 + lr, (2 * ndp + (mi >> 1)) * 8));
      mma_16816<T>(o[2 * ndp], pa, b[0], b[1]);
      mma_16816<T>(o[2 * ndp + 1], pa, b[2], b[3]);
    }
  }

  // this warp's O [group][D], maxima and sums to shared memory
  __device__ __forceinline__ void store(float *mo, float *mm, float *ml, int group) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    l_run += __shfl_xor_sync(kFull, l_run, 1);
    l_run += __shfl_xor_sync(kFull, l_run, 2);
    if (gid >= group) return;
#pragma unroll
    for (int nd = 0; nd < NTD; ++nd)
      *reinterpret_cast<float2 *>(mo + gid * D + nd * 8 + 2 * tig) =
          make_float2(o[nd][0] * (1.f / kScaleP), o[nd][1] * (1.f / kScaleP));
    if (tig == 0) {
      mm[gid] = m_run;
      ml[gid] = l_run;
    }
  }
};

// ---- one page of one kv head: f32 on the FMA pipe ---------------------------------------
template <int D_, int G> struct PageF32 {
  using T = float;
  static constexpr int D = D_, WARPS = 4, NSTAGE = D == 128 ? 1 : 2;
  static constexpr int DPL = D / 32, TILE = kBS * D, TILE_BYTES = TILE * 4;
  static constexpr int SUB = (G > 4) ? 8 : 16;  // tokens per scoring sub-tile
  static constexpr int NV = G * SUB, NVP = ((NV + 31) / 32) * 32;
  static constexpr int R = NVP / 32;   // totals per lane after the butterfly
  static constexpr int LPH = SUB / R;  // lanes per head
  static_assert(LPH * R == SUB && LPH * G <= 32, "lane mapping");
  float qv[G][DPL], acc[G][DPL], m_run[G];
  float l_lane = 0.f;

  __device__ __forceinline__ void init(const float *q, int, float qscale) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < G; ++h) {
      TileLoad<float, D>::load(q + h * D, lane, qv[h]);
      m_run[h] = kLowest;
#pragma unroll
      for (int d = 0; d < DPL; ++d) {
        qv[h][d] *= qscale;
        acc[h][d] = 0.f;
      }
    }
  }

  static __device__ __forceinline__ void issue(unsigned char *st, const CUtensorMap &, const CUtensorMap &,
                                               const RowsParams &p, int page, int kvh, int hkv, uint64_t *bar) {
    const size_t at = (size_t(page) * hkv + kvh) * TILE;
    mbar_expect_tx(bar, 2 * TILE_BYTES);
    bulk_g2s(st, static_cast<const float *>(p.k_pool) + at, TILE_BYTES, bar);
    bulk_g2s(st + TILE_BYTES, static_cast<const float *>(p.v_pool) + at, TILE_BYTES, bar);
  }

  __device__ __forceinline__ void page(unsigned char *st, uint32_t bits, float, float *raw, int raw_stride, int) {
    const int lane = threadIdx.x & 31;
    const float *kt = reinterpret_cast<const float *>(st), *vt = kt + TILE;
    const int hl = lane / LPH;  // head of this lane's score totals (>= G: padding lane)
#pragma unroll
    for (int t0 = 0; t0 < kBS; t0 += SUB) {
      const uint32_t live = bits >> t0 & ((1u << SUB) - 1);  // warp-uniform
      if (!live) {
        if (raw && hl < G)
#pragma unroll
          for (int j = 0; j < R; ++j) raw[size_t(hl) * raw_stride + t0 + (lane * R + j) % SUB] = -INFINITY;
        continue;
      }
      float v[NVP];
#pragma unroll
      for (int i = 0; i < NVP; ++i) v[i] = 0.f;
#pragma unroll
      for (int t = 0; t < SUB; ++t) {
        if (live >> t & 1) {
          float kk[DPL];
          TileLoad<float, D>::load(kt + (t0 + t) * D, lane, kk);
#pragma unroll
          for (int h = 0; h < G; ++h) {
            float a = 0.f;
#pragma unroll
            for (int d = 0; d < DPL; ++d) a = fmaf(qv[h][d], kk[d], a);
            v[h * SUB + t] = a;
          }
        }
      }
      Butterfly<NVP, 16>::run(v, lane);
      // lane holds totals for index lane * R + j -> head hl, token (lane * R + j) % SUB
      float mloc = -INFINITY;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int t = (lane * R + j) % SUB;
        if (hl >= G || !(live >> t & 1)) v[j] = -INFINITY;
        if (raw && hl < G) raw[size_t(hl) * raw_stride + t0 + t] = v[j];
        mloc = fmaxf(mloc, v[j]);
      }
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) mloc = fmaxf(mloc, __shfl_xor_sync(kFull, mloc, o));
      float alpha[G], mh = -INFINITY, al = 1.f;
#pragma unroll
      for (int h = 0; h < G; ++h) {
        const float mn = fmaxf(m_run[h], __shfl_sync(kFull, mloc, h * LPH));
        alpha[h] = exp2f(m_run[h] - mn);
        m_run[h] = mn;
        if (hl == h) {
          mh = mn;
          al = alpha[h];
        }
      }
      float pv[R], psum = 0.f;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        pv[j] = (v[j] == -INFINITY) ? 0.f : exp2f(v[j] - mh);
        psum += pv[j];
      }
      l_lane = l_lane * al + psum;
#pragma unroll
      for (int h = 0; h < G; ++h)
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[h][d] *= alpha[h];
#pragma unroll
      for (int t = 0; t < SUB; ++t) {
        if (live >> t & 1) {
          float vv[DPL];
          TileLoad<float, D>::load(vt + (t0 + t) * D, lane, vv);
#pragma unroll
          for (int h = 0; h < G; ++h) {
            const int idx = h * SUB + t;
            const float ph = __shfl_sync(kFull, pv[idx % R], idx / R);
#pragma unroll
            for (int d = 0; d < DPL; ++d) acc[h][d] = fmaf(ph, vv[d], acc[h][d]);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void store(float *mo, float *mm, float *ml, int) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) l_lane += __shfl_xor_sync(kFull, l_lane, o);
#pragma unroll
    for (int h = 0; h < G; ++h) {
#pragma unroll
      for (int d = 0; d < DPL; ++d) mo[h * D + lane * DPL + d] = acc[h][d];
      const float lh = __shfl_sync(kFull, l_lane, h * LPH);
      if (lane == 0) {
        mm[h] = m_run[h];
        ml[h] = lh;
      }
    }
  }
};

constexpr int kMaxGroup = 8;

// Page::D * kMaxGroup floats for each warp's O and the CTA's; the maxima and sums of both
template <class Page> struct Layout {
  static constexpr int W = Page::WARPS;
  static constexpr size_t kStages = size_t(W) * Page::NSTAGE * 2 * Page::TILE_BYTES;
  static constexpr size_t kBars = W * Page::NSTAGE * sizeof(uint64_t);
  static constexpr size_t kMerge = (size_t(W) + 1) * kMaxGroup * (Page::D + 2) * sizeof(float);
  static constexpr size_t kSmem = 1024 + std::max(kStages + kBars, kMerge);
};

template <class Page, bool WEIGHTS>
__global__ void __launch_bounds__(Page::WARPS * 32)
    window_rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       RowsParams p, int C) {
  constexpr int W = Page::WARPS, NSTAGE = Page::NSTAGE, STAGE_BYTES = 2 * Page::TILE_BYTES, D = Page::D;
  using T = typename Page::T;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char *smem =
      reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + Layout<Page>::kStages);

  const int ri = blockIdx.x / C, part = blockIdx.x % C;  // part = rank in the cluster
  const int row = p.row_index ? p.row_index[ri] : ri;
  const int kvh = blockIdx.y, G = p.group;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int ctx = p.row_ctx[row];
  const int trow = ctx == 0 ? 0 : p.row_table ? p.row_table[row] : row;  // an empty row names none
  bool ok = ctx >= 0 && ctx <= p.max_ctx && trow >= 0 && trow < p.table_rows;
  if (WEIGHTS && table_row_repeated(p.row_table, p.row_ctx, row, trow) && ctx != 0) ok = false;
  if (!ok) {  // the whole cluster leaves
    if (t == 0) atomicOr(p.status, kStatusBadIndex);
    return;
  }
  const int32_t *table = p.block_tables + size_t(trow) * p.max_blocks_per_seq;
  const int low = VisiblePages::lowest_key(ctx - 1, p.window);
  const VisiblePages vis(ctx - 1, ctx, p.window, p.sinks);
  const int share = (vis.count + C - 1) / C;
  const int b0 = min(part * share, vis.count), b1 = min(b0 + share, vis.count);
  const int nb_w = (b1 - b0 - warp + W - 1) / W;  // pages b0 + warp + k * W
  unsigned char *my_stage = smem + size_t(warp) * NSTAGE * STAGE_BYTES;
  uint64_t *my_bar = bars + warp * NSTAGE;
  if (lane == 0) {
    for (int s = 0; s < NSTAGE; ++s) mbar_init(&my_bar[s], 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  __syncwarp();

  int page_reg = 0;  // lane k holds the page id of this warp's k-th page (32 at a time)
  auto page_of = [&](int k) -> int { return __shfl_sync(kFull, page_reg, k & 31); };
  auto refill_pages = [&](int k0) {
    const int k = k0 + lane;
    page_reg = 0;
    if (k < nb_w) {
      const int page = table[vis.page_at(b0 + warp + k * W)];
      if (page >= 0 && page < p.pool_blocks) page_reg = page;
      else atomicOr(p.status, kStatusBadIndex);
    }
  };
  auto issue = [&](int s, int page) {
    if (lane == 0)
      Page::issue(my_stage + size_t(s) * STAGE_BYTES, kmap, vmap, p, page, kvh, p.num_kv_heads, &my_bar[s]);
  };
  bool failed = false;
  int issued = 0, kfail = 0;
  if (nb_w > 0) {
    refill_pages(0);
    const int pro = min(NSTAGE, nb_w);
    for (int k = 0; k < pro; ++k) issue(k, page_of(k));
    issued = pro;
  }
  Page pg;
  const size_t head0 = (size_t(row) * p.num_kv_heads + kvh) * G;
  pg.init(static_cast<const T *>(p.q) + head0 * D, G, p.qscale);
  float *raw = WEIGHTS ? p.raw + head0 * p.ctx16 : nullptr;

  for (int k = 0; k < nb_w; ++k) {
    const int s = k % NSTAGE;
    // the whole warp agrees before leaving, so no lane is left waiting in a shuffle
    if (!__all_sync(kFull, mbar_wait_bounded(&my_bar[s], (k / NSTAGE) & 1, p.wait_limit))) {
      failed = true;
      kfail = k;
      break;
    }
    const int key0 = vis.page_at(b0 + warp + k * W) * kBS;
    const uint32_t bits =
        0xffffu & low_bits(ctx - key0) & (~low_bits(low - key0) | low_bits(p.sinks - key0));
    pg.page(my_stage + size_t(s) * STAGE_BYTES, bits, p.qscale, WEIGHTS ? raw + key0 : nullptr, p.ctx16, G);
    __syncwarp();
    if (issued < nb_w && k + NSTAGE == issued) {
      const int kn = issued;
      if ((kn & 31) == 0) refill_pages(kn);
      const int page = page_of(kn);
      if (lane == 0) fence_proxy_async();
      issue(s, page);
      ++issued;
    }
  }
  if (failed) {
    if (lane == 0) atomicOr(p.status, kStatusWaitTimeout);
    for (int k = kfail; k < issued; ++k) mbar_wait_bounded(&my_bar[k % NSTAGE], (k / NSTAGE) & 1);
  }

  // ---- merge the warps (the stages are free), then the cluster's CTAs ----
  float *wo = reinterpret_cast<float *>(smem);         // [W][kMaxGroup][D]
  float *wm = wo + W * kMaxGroup * D;                  // [W][kMaxGroup] maxima, then the row's
  float *wl = wm + W * kMaxGroup;                      // and sums, then the row's reciprocal
  float *co = wl + W * kMaxGroup;                      // the CTA's [G][D], maxima, sums
  float *cm = co + kMaxGroup * D, *cl = cm + kMaxGroup;
  const bool any_failed = __syncthreads_or(failed ? 1 : 0) != 0;
  pg.store(wo + warp * kMaxGroup * D, wm + warp * kMaxGroup, wl + warp * kMaxGroup, G);
  __syncthreads();
  T *out = static_cast<T *>(p.out) + head0 * D;
  for (int i = t; i < G * D; i += W * 32) {
    const int h = i / D;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, wm[w * kMaxGroup + h]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = exp2f(wm[w * kMaxGroup + h] - M);
      L += f * wl[w * kMaxGroup + h];
      O += f * wo[w * kMaxGroup * D + i];
    }
    // (a row that sees no key has L = 0; a NaN that it sees makes L NaN, and its result)
    if (C == 1 && !any_failed) out[i] = Elem<T>::from_f(L == 0.f ? 0.f : O / L);
    co[i] = O;
    if (i % D == 0) {
      cm[h] = any_failed ? NAN : M;  // a NaN maximum tells the cluster that a wait ran out (fmaxf gives none)
      cl[h] = L;
    }
  }
  // All CTAs' maxima and sums, one load a thread; then each head's maximum and the CTAs' factors
  // 2^(m_c - M) / L (the warps' O is free by now).
  float *tm = wo, *tl = tm + kMaxCluster * kMaxGroup, *tf = tl + kMaxCluster * kMaxGroup;  // [CTA][kMaxGroup]
  if (C > 1) {
    cluster_sync();
    for (int i = t; i < C * kMaxGroup; i += W * 32) {
      const int c = i / kMaxGroup, h = i % kMaxGroup;
      if (h < G) {
        tm[i] = peer_f32(cm + h, c);
        tl[i] = peer_f32(cl + h, c);
      }
    }
  } else if (WEIGHTS) {
    __syncthreads();
    if (t < G) {
      tm[t] = cm[t];
      tl[t] = cl[t];
    }
  }
  if (C > 1 || WEIGHTS) {
    __syncthreads();
    if (t < G) {
      float M = -INFINITY, L = 0.f;
      bool bad = false;
      for (int c = 0; c < C; ++c) {
        const float mc = tm[c * kMaxGroup + t];
        bad |= mc != mc;
        M = fmaxf(M, mc);
      }
      for (int c = 0; c < C; ++c) {
        const float f = exp2f(tm[c * kMaxGroup + t] - M);
        tf[c * kMaxGroup + t] = f;
        L += f * tl[c * kMaxGroup + t];
      }
      wm[t] = bad ? NAN : M;
      wl[t] = L == 0.f ? 0.f : 1.f / L;
    }
    __syncthreads();
  }
  const bool good = (C == 1 && !WEIGHTS) || wm[0] == wm[0];
  if (C > 1 && good)
    for (int i = part * W * 32 + t; i < G * D; i += C * W * 32) {
      const int h = i / D;
      float o[kMaxCluster], O = 0.f;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) o[c] = c < C ? peer_f32(co + i, c) : 0.f;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c)
        if (c < C) O += tf[c * kMaxGroup + h] * o[c];
      out[i] = Elem<T>::from_f(O * wl[h]);
    }
  if (C > 1) cluster_arrive();
  if constexpr (WEIGHTS) {
    float *sum = p.weight_sum + (size_t(trow) * p.num_kv_heads + kvh) * p.weight_stride;
    // 4 keys a thread, all heads' scores and the sums under way together: the CTA streams nothing
    // meanwhile (a key at a time this phase took a fifth of the kernel)
    const int end = good ? min(b1 * kBS, ctx) : 0;
    const bool vec = (reinterpret_cast<uintptr_t>(sum) & 15) == 0;
    for (int key = b0 * kBS + 4 * t; key < end; key += 4 * W * 32) {
      float4 r[kMaxGroup];
#pragma unroll
      for (int h = 0; h < kMaxGroup; ++h)
        if (h < G) r[h] = *reinterpret_cast<const float4 *>(raw + size_t(h) * p.ctx16 + key);
      const bool whole = vec && key + 4 <= end;
      float s[4];
      if (whole) {
        Vec4<float>::load(sum + key, s);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = key + i < end ? sum[key + i] : 0.f;
      }
      float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < kMaxGroup; ++h)
        if (h < G) {
          const float m = wm[h], f = wl[h];
          add[0] += exp2f(r[h].x - m) * f;
          add[1] += exp2f(r[h].y - m) * f;
          add[2] += exp2f(r[h].z - m) * f;
          add[3] += exp2f(r[h].w - m) * f;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += add[i];
      if (whole) {
        Vec4<float>::store(sum + key, s);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key + i < end) sum[key + i] = s[i];
      }
    }
  }
  if (C > 1) cluster_wait();  // no CTA leaves while another may read its shared memory
}

// CTAs per (row, kv head); `slots`: CTAs that the machine holds at once.  Fewer pairs than slots
// are split to fill one wave (12 rows x 4 heads of 16k keys with weights: 8 CTAs each 70 us, 1 each
// 243 us), down to two pages a warp and to a cluster of 8 (16, the most there is, measured slower
// for one row: 7.1 against 6.6 us).  Between one and four waves of whole rows, halves even out
// ragged lengths (64 rows x 8 heads: 154 against 169 us); more rows do that by themselves.
int cluster_size(int rows, int hkv, int max_pages, int warps, int slots) {
  const long long pairs = (long long)rows * hkv;
  long long c = pairs > slots ? (pairs < 4 * slots ? 2 : 1) : slots / pairs;
  c = std::min<long long>(c, kMaxCluster);
  return int(std::max<long long>(1, std::min<long long>(c, max_pages / (2 * warps))));
}

template <class Page, bool WEIGHTS>
cudaError_t launch_rows(const RowsParams &p, int rows, int max_pages, const CUtensorMap &km, const CUtensorMap &vm,
                        cudaStream_t stream) {
  auto kern = window_rows_kernel<Page, WEIGHTS>;
  static std::atomic<bool> attr_done[64];  // per device; zero-initialised (static storage)
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Layout<Page>::kSmem));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_done[dev].store(true, std::memory_order_release);  // setting twice is harmless
  }
  const int slots = 148 * int(std::min<size_t>(227 * 1024 / (Layout<Page>::kSmem + 1024), 16));
  const int C = cluster_size(rows, p.num_kv_heads, max_pages, Page::WARPS, slots);
  if ((long long)rows * C > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(rows) * C, p.num_kv_heads);
  cfg.blockDim = dim3(Page::WARPS * 32);
  cfg.dynamicSmemBytes = Layout<Page>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = C;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, km, vm, p, C);
}

template <class Page>
cudaError_t launch_page(const RowsParams &p, int rows, int max_pages, const CUtensorMap &km, const CUtensorMap &vm,
                        cudaStream_t stream) {
  return p.weight_sum ? launch_rows<Page, true>(p, rows, max_pages, km, vm, stream)
                      : launch_rows<Page, false>(p, rows, max_pages, km, vm, stream);
}

template <int D>
cudaError_t launch_f32(const RowsParams &p, int rows, int max_pages, cudaStream_t stream) {
  const CUtensorMap none{};
  switch (p.group) {
    case 1: return launch_page<PageF32<D, 1>>(p, rows, max_pages, none, none, stream);
    case 2: return launch_page<PageF32<D, 2>>(p, rows, max_pages, none, none, stream);
    case 4: return launch_page<PageF32<D, 4>>(p, rows, max_pages, none, none, stream);
    case 7: return launch_page<PageF32<D, 7>>(p, rows, max_pages, none, none, stream);
    case 8: return launch_page<PageF32<D, 8>>(p, rows, max_pages, none, none, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_checked(const WindowArgs &a, cudaStream_t stream) {
  RowsParams p{};
  p.q = a.q;
  p.k_pool = a.k_pool;
  p.v_pool = a.v_pool;
  p.block_tables = a.block_tables;
  p.row_table = a.row_table;
  p.row_ctx = a.row_ctx;
  p.row_index = a.row_index;
  p.out = a.out;
  p.weight_sum = a.weight_sum;
  p.raw = static_cast<float *>(a.workspace);
  p.weight_stride = a.weight_stride;
  p.pool_blocks = int(a.pool_blocks);  // < 2^31 (pools_ok)
  p.table_rows = a.table_rows;
  p.max_blocks_per_seq = a.max_blocks_per_seq;
  p.max_ctx = a.max_ctx;
  p.ctx16 = (a.max_ctx + kBS - 1) / kBS * kBS;
  p.window = a.window;
  p.sinks = a.sinks;
  p.num_kv_heads = a.num_kv_heads;
  p.group = a.num_heads / a.num_kv_heads;
  p.qscale = a.scale * kLog2e;
  p.wait_limit = page_wait_limit();
  p.status = a.status;
  if (!p.status) {
    const cudaError_t e = standalone_status_word(&p.status);
    if (e != cudaSuccess) return e;
  }
  // by the window where there is one, not by this call's contexts: a row's result does not
  // change with the longest context it is batched with
  const int64_t most = a.window > 0 ? int64_t(a.window) + a.sinks : a.max_ctx;
  const int max_pages = int(std::min<int64_t>(most / kBS + 2, 1 << 26));
  if (a.dtype == MS_DTYPE_F32)
    return a.head_dim == 128 ? launch_f32<128>(p, a.num_rows, max_pages, stream) : launch_f32<64>(p, a.num_rows, max_pages, stream);
  CUtensorMap km, vm;
  const int64_t tiles = a.pool_blocks * a.num_kv_heads;
  if (a.k_map && a.v_map) {
    km = *static_cast<const CUtensorMap *>(a.k_map);
    vm = *static_cast<const CUtensorMap *>(a.v_map);
  } else if (!encode_pool_tensor_map(&km, a.k_pool, a.dtype, a.head_dim, tiles) ||
             !encode_pool_tensor_map(&vm, a.v_pool, a.dtype, a.head_dim, tiles)) {
    return cudaErrorInvalidValue;
  }
  if (a.dtype == MS_DTYPE_BF16)
    return a.head_dim == 128 ? launch_page<PageTc<__nv_bfloat16, 128>>(p, a.num_rows, max_pages, km, vm, stream)
                             : launch_page<PageTc<__nv_bfloat16, 64>>(p, a.num_rows, max_pages, km, vm, stream);
  return a.head_dim == 128 ? launch_page<PageTc<__half, 128>>(p, a.num_rows, max_pages, km, vm, stream)
                           : launch_page<PageTc<__half, 64>>(p, a.num_rows, max_pages, km, vm, stream);
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
  if (!common_ok(a) || !ptr4(a.row_ctx) || a.tiles || a.max_ctx > int64_t(a.max_blocks_per_seq) * attn::kBS ||
      (a.row_table ? !ptr4(a.row_table) : a.table_rows < a.num_rows))
    return cudaErrorInvalidValue;
  if (a.weight_sum) {
    const int64_t need = attention_weights_workspace_bytes(a.num_rows, a.num_heads, a.max_ctx);
    if (a.row_index || !ptr4(a.weight_sum) || a.weight_stride < a.max_ctx || (need > 0 && !ptr16(a.workspace)) || a.workspace_bytes < need)
      return cudaErrorInvalidValue;
  }
  return launch_checked(a, stream);
}

cudaError_t launch_window_prefill(const WindowArgs &args, cudaStream_t stream) {
  WindowArgs a = args;
  if (a.num_tiles < 0) return cudaErrorInvalidValue;
  if (a.num_tiles == 0) return cudaSuccess;
  if (!common_ok(a) || !ptr4(a.tiles) || a.dtype == MS_DTYPE_F32 || a.num_tiles > 65535) return cudaErrorInvalidValue;
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
