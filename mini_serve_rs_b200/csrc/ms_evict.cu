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
// Two launches.  The first selects: a cluster of C CTAs serves one (sequence, kv
// head); each holds a run of slots, their 32-bit rank keys (whose unsigned order
// is the order of the weights; protected slots: the largest key) in shared
// memory.
//  1. T, the keep-th largest key, by a radix search of three digits from the
//     top (11, 11 and 10 bits): histogram of the keys that match the digits
//     found so far, summed over the cluster through distributed shared memory,
//     and the digit in which the keep-th largest lies.  It ends early where
//     all keys with T's digits so far stay.
//  2. Slots above T stay, and of the slots equal to T the lowest that still
//     fit: one bit each.  Counts of holes and movers per word, scanned over the
//     CTA and the cluster, give each its rank; the lists of holes and movers
//     and their length go to the workspace.
// The second moves: 8 moves a warp (256-byte rows), all of a call's moves at
// once on as many warps, because a row in a large pool costs a long latency
// (address translation included) and few bytes: with the moves left to the CTA
// that selected them, 8 at a time per warp, the longest sequences of a ragged
// batch finished long after the others (64 sequences: 68 us against 44).
// Latency-bound for one sequence (a chain of loads and barriers), bound by the
// moves' HBM traffic for many.
#include <algorithm>
#include <atomic>
#include <cstddef>

#include "ms_window.cuh"

namespace ms {
namespace {

using attn::kBS;

constexpr int kMaxCluster = 8;
constexpr int kMaxSlots = 32768;  // rank keys of one CTA in shared memory
constexpr int kDigits = 3;
constexpr int kBins = 2048;

struct EvictParams {
  unsigned char *k_pool, *v_pool;
  int64_t pool_blocks;
  const int32_t *block_tables;
  int table_rows, max_blocks_per_seq;
  const int32_t *row_table, *row_ctx, *row_next, *row_known;
  int max_ctx, keep, sinks, recent;
  const float *w_in;
  float *w_out;
  const int32_t *pos_in;
  int32_t *pos_out;
  int64_t stride;
  int num_kv_heads;
  int chunks;      // 16-byte pieces of one K (V) row
  int vec;         // weights and positions may be read and written 16 bytes at a time
  int32_t *lists;  // [rows][kv heads][2][half]: holes, movers
  int half;
  int32_t *moves;  // [rows][kv heads]: their number
  unsigned *status;
};

// unsigned order of the result = order of the weights; -0 as 0, every NaN above infinity
__device__ __forceinline__ uint32_t rank_key(float w) {
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct alignas(16) Shared {  // histograms and slices are read 16 bytes at a time
  uint32_t hist[kDigits][kBins];  // of each digit (read by the cluster)
  uint32_t slice[kBins / 2];      // the cluster's sum of the bins this CTA adds up (read by the cluster)
  uint32_t warp_sum[32];
  uint32_t counts[2];             // this CTA's equal slots; holes | movers << 16 (read by the cluster)
  uint32_t digit;
  int left, equal;
};
static_assert(alignof(Shared) == 16 && offsetof(Shared, slice) % 16 == 0 && sizeof(Shared) % 16 == 0,
              "16-byte accesses; the dynamic part may follow it");

// sum of v over the threads before this one; the CTA's total in `all`.  `scratch` is free again
// after the next barrier.
template <int NT>
__device__ __forceinline__ uint32_t scan_before(uint32_t v, uint32_t *scratch, uint32_t &all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(kFull, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) scratch[warp] = s;
  __syncthreads();
  const uint32_t c = lane < NT / 32 ? scratch[lane] : 0;
  all = __reduce_add_sync(kFull, c);
  return __reduce_add_sync(kFull, lane < warp ? c : 0u) + s - v;
}

// The digit in which the keep-th largest value lies, counted from the top, over the cluster's
// histograms of digit d (complete in shared memory): into sh.digit, sh.left (what is left to
// find inside it) and sh.equal (the values in it), behind a barrier.
template <int NT>
__device__ __forceinline__ void find_digit(Shared &sh, int d, int C, int keep) {
  constexpr int B = kBins / NT;  // bins of a thread, the largest digits first
  const int t = threadIdx.x, b0 = kBins - B * (t + 1);
  uint32_t c[B];
  // CTA r adds up the r-th of C slices of the bins, then everyone takes the sums from their
  // owners: 2 x 8 KB of distributed shared memory per CTA instead of C x 8 KB
  const int slice = kBins / C;
  if (C > 1) {
    const int own = int(blockIdx.x % C) * slice;
    for (int i = 4 * t; i < slice; i += 4 * NT) {
      uint4 v = make_uint4(0, 0, 0, 0);
      for (int r = 0; r < C; ++r) {
        const uint4 u = peer_u4(&sh.hist[d][own + i], r);
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
      }
      *reinterpret_cast<uint4 *>(&sh.slice[i]) = v;
    }
    cluster_sync();
  }
#pragma unroll
  for (int i = 0; i < B; i += 4) {
    const int b = b0 + i;
    const uint4 v = C == 1 ? *reinterpret_cast<const uint4 *>(&sh.hist[d][b]) : peer_u4(&sh.slice[b % slice], b / slice);
    c[i] = v.x;
    c[i + 1] = v.y;
    c[i + 2] = v.z;
    c[i + 3] = v.w;
  }
  uint32_t sum = 0, all;
#pragma unroll
  for (int i = 0; i < B; ++i) sum += c[i];
  uint32_t above = scan_before<NT>(sum, sh.warp_sum, all);
  if (above < uint32_t(keep) && above + sum >= uint32_t(keep)) {  // one thread
#pragma unroll
    for (int i = B - 1; i >= 0; --i) {
      if (above < uint32_t(keep) && above + c[i] >= uint32_t(keep)) {
        sh.digit = b0 + i;
        sh.left = keep - int(above);
        sh.equal = int(c[i]);
      }
      above += c[i];
    }
  }
  __syncthreads();
}

// the n lowest set bits of w
__device__ __forceinline__ uint32_t lowest_bits(uint32_t w, int n) {
  if (n >= __popc(w)) return w;
  uint32_t out = 0;
  for (; n > 0; --n) {
    out |= w & (0u - w);
    w &= w - 1;
  }
  return out;
}

// Moves [r0, r0 + moves_per_warp()) of one head, as far as there are `count`, by one warp: a lane
// each looks up the pages and takes the mover's weight and position along, then their K and V
// rows are copied, every load before the first store.  jt, jf: the lane's hole and mover.
__device__ __forceinline__ int moves_per_warp(const EvictParams &p) { return 4 * (32 / p.chunks); }
__device__ __forceinline__ void move_rows(const EvictParams &p, int row, int h, int jt, int jf, int count) {
  const int lane = threadIdx.x & 31;
  const int per = 32 / p.chunks, sub = lane / p.chunks, ch = lane % p.chunks;  // chunks: 8, 16 or 32
  long long to = -1, from = -1;  // row of the pool, -1 where there is nothing to copy
  if (lane < min(count, 4 * per)) {
    const int n = p.row_ctx[row], trow = p.row_table ? p.row_table[row] : row;
    const int known = p.row_known ? p.row_known[row] : 0;
    const int32_t *table = p.block_tables + size_t(trow) * p.max_blocks_per_seq;
    const int pt = table[jt / kBS], pf = table[jf / kBS];
    const size_t base = (size_t(trow) * p.num_kv_heads + h) * size_t(p.stride);
    const float w = p.w_in[base + jf];
    const int pos = jf < known ? p.pos_in[base + jf] : p.row_next[row] - n + jf;
    if (pt >= 0 && pt < p.pool_blocks && pf >= 0 && pf < p.pool_blocks) {
      to = ((long long)(pt) * p.num_kv_heads + h) * kBS + jt % kBS;
      from = ((long long)(pf) * p.num_kv_heads + h) * kBS + jf % kBS;
    } else {
      atomicOr(p.status, kStatusBadIndex);
    }
    p.w_out[base + jt] = w;
    p.w_out[base + jf] = 0.f;  // after it was read: weight_out may be weight_in
    p.pos_out[base + jt] = pos;
  }
  uint4 kv[4], vv[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const long long src = __shfl_sync(kFull, from, u * per + sub);
    if (src >= 0) {
      kv[u] = reinterpret_cast<const uint4 *>(p.k_pool)[src * p.chunks + ch];
      vv[u] = reinterpret_cast<const uint4 *>(p.v_pool)[src * p.chunks + ch];
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const long long dst = __shfl_sync(kFull, to, u * per + sub);
    if (dst >= 0) {
      reinterpret_cast<uint4 *>(p.k_pool)[dst * p.chunks + ch] = kv[u];
      reinterpret_cast<uint4 *>(p.v_pool)[dst * p.chunks + ch] = vv[u];
    }
  }
}

// FUSED: the cluster's warps also make the moves.
template <int NT, bool FUSED>
__global__ void __launch_bounds__(NT, 1024 / NT) evict_kernel(EvictParams p, int C, int seg) {
  constexpr int kWarpsNT = NT / 32;
  // [seg] rank keys, then [seg / 32] words three times
  extern __shared__ __align__(16) uint32_t keys[];  // (written four at a time)
  uint32_t *stay = keys + seg;        // slots above T, then slots that stay, one bit each
  uint32_t *equal_w = stay + seg / 32;  // slots equal to T, then movers before each word
  uint32_t *hole0 = equal_w + seg / 32;  // holes before each word
  __shared__ Shared sh;
  const int row = blockIdx.x / C, part = blockIdx.x % C, h = blockIdx.y;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int n = p.row_ctx[row], next = p.row_next[row];
  const int trow = n == 0 ? 0 : p.row_table ? p.row_table[row] : row;  // an empty row names none
  const int known = p.row_known ? p.row_known[row] : 0;
  for (int i = t; i < kDigits * kBins / 4; i += NT)
    reinterpret_cast<uint4 *>(sh.hist)[i] = make_uint4(0, 0, 0, 0);
  bool ok = n == 0 || (n > 0 && n <= p.max_ctx && trow >= 0 && trow < p.table_rows && known >= 0 && next >= n);
  if (table_row_repeated(p.row_table, p.row_ctx, row, trow) && n != 0) ok = false;  // (with a barrier)
  const size_t pair = size_t(row) * p.num_kv_heads + h;
  if (!ok) {  // the whole cluster leaves
    if (t == 0) {
      atomicOr(p.status, kStatusBadIndex);
      if (part == 0) p.moves[pair] = 0;
    }
    return;
  }
  const size_t base = (size_t(trow) * p.num_kv_heads + h) * size_t(p.stride);
  const float *w_in = p.w_in + base;
  float *w_out = p.w_out + base;
  const int32_t *pos_in = p.pos_in ? p.pos_in + base : nullptr;
  int32_t *pos_out = p.pos_out + base;
  auto position = [&](int j) { return j < known ? pos_in[j] : next - n + j; };
  const int s0 = part * seg, s1 = min(s0 + seg, n), len = max(0, s1 - s0);  // this CTA's slots
  if (n <= p.keep) {  // nothing to evict
    if (part == 0 && t == 0) p.moves[pair] = 0;
    for (int j = s0 + t; j < s1; j += NT) {
      w_out[j] = w_in[j];
      pos_out[j] = position(j);
    }
    return;
  }

  // ---- 1. the keep-th largest key ----
  // Slots go four to a thread here and in the last step, as vectors where the arrays allow it
  // (p.vec; a slot index is a multiple of 4 and the stride too, so a vector never leaves its row),
  // U of them under way before the first is used: these two steps are loads' latency.
  constexpr int U = 3;
  auto load_weights = [&](int j, float (&w)[4]) {
    if (p.vec) {
      Vec4<float>::load(w_in + j, w);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = j + i < s1 ? w_in[j + i] : 0.f;
    }
  };
  auto load_positions = [&](int j, int (&pos)[4]) {
    if (p.vec && j + 4 <= known) {
      const int4 v = *reinterpret_cast<const int4 *>(pos_in + j);
      pos[0] = v.x, pos[1] = v.y, pos[2] = v.z, pos[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) pos[i] = j + i < s1 ? position(j + i) : 0;
    }
  };
  for (int j0 = s0 + 4 * t; j0 < s1; j0 += U * 4 * NT) {
    float w[U][4];
    int pos[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j0 + u * 4 * NT < s1) {
        load_weights(j0 + u * 4 * NT, w[u]);
        load_positions(j0 + u * 4 * NT, pos[u]);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * 4 * NT;
      if (j >= s1) break;
      uint32_t key[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        key[i] = pos[u][i] < p.sinks || pos[u][i] >= next - p.recent ? 0xffffffffu : rank_key(w[u][i]);
        if (j + i < s1) atomicAdd(&sh.hist[0][key[i] >> 21], 1u);
      }
      *reinterpret_cast<uint4 *>(keys + j - s0) = make_uint4(key[0], key[1], key[2], key[3]);  // (seg: a multiple of 32)
    }
  }
  uint32_t T = 0;
  int left = p.keep, equal = 0;  // of the keys with T's digits so far: to keep, and in all
#pragma unroll
  for (int d = 0; d < kDigits; ++d) {
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
    if (d > 0) {
      const int up = d == 1 ? 21 : 10;
      const uint32_t mask = d == 1 ? 2047u : 1023u;
#pragma unroll 4
      for (int j = t; j < len; j += NT) {
        const uint32_t key = keys[j];
        if (key >> up == T >> up) atomicAdd(&sh.hist[d][key >> shift & mask], 1u);
      }
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    find_digit<NT>(sh, d, C, left);
    T |= sh.digit << shift;
    left = sh.left;
    equal = sh.equal;
    if (left == equal) break;  // all of them stay: T's other digits may be 0 (the same for the cluster)
  }

  // ---- 2. which slots stay; holes and movers in order ----
  const bool all_equal = left == equal;  // key >= T stays; else key > T, and the lowest `left` equal ones
  const int words = (len + 31) / 32;
  for (int i = warp; i < words; i += kWarpsNT) {
    const int j = i * 32 + lane;
    const uint32_t key = j < len ? keys[j] : 0u;
    const unsigned gt = __ballot_sync(kFull, j < len && (all_equal ? key >= T : key > T));
    const unsigned eq = __ballot_sync(kFull, j < len && key == T);
    if (lane == 0) {
      stay[i] = gt;
      equal_w[i] = eq;
    }
  }
  __syncthreads();
  // thread t takes words [t q, t q + q): ranks follow the slot order
  const int q = (seg / 32 + NT - 1) / NT;
  const int wa = min(t * q, words), wb = min(wa + q, words);
  if (!all_equal) {
    uint32_t c = 0, all;
    for (int i = wa; i < wb; ++i) c += __popc(equal_w[i]);
    int tie = int(scan_before<NT>(c, sh.warp_sum, all));
    if (C > 1) {
      if (t == 0) sh.counts[0] = all;
      cluster_sync();
      for (int r = 0; r < part; ++r) tie += int(peer_u32(&sh.counts[0], r));
    }
    for (int i = wa; i < wb; ++i) {
      const uint32_t eq = equal_w[i];
      stay[i] |= lowest_bits(eq, left - tie);
      tie += __popc(eq);
    }
    __syncthreads();  // warp_sum is used again
  }
  auto below_keep = [&](int i) { return low_bits(p.keep - s0 - 32 * i); };  // slots of word i that are below keep
  auto live = [&](int i) { return low_bits(len - 32 * i); };
  uint32_t cnt = 0, all;
  for (int i = wa; i < wb; ++i)
    cnt += __popc(live(i) & below_keep(i) & ~stay[i]) + (__popc(stay[i] & ~below_keep(i)) << 16);
  const uint32_t rank = scan_before<NT>(cnt, sh.warp_sum, all);
  int rank_h = rank & 0xffff, rank_m = rank >> 16, moves = all >> 16;
  if (C > 1) {
    if (t == 0) sh.counts[1] = all;
    cluster_sync();
    moves = 0;
    for (int r = 0; r < C; ++r) {
      const uint32_t c = peer_u32(&sh.counts[1], r);
      if (r < part) {
        rank_h += c & 0xffff;
        rank_m += c >> 16;
      }
      moves += c >> 16;
    }
  }
  if (part == 0 && t == 0) p.moves[pair] = moves;
  int32_t *holes = p.lists + pair * 2 * size_t(p.half), *movers = holes + p.half;
  for (int i = wa; i < wb; ++i) {
    const uint32_t s = stay[i], lo = below_keep(i);
    equal_w[i] = rank_m;
    hole0[i] = rank_h;
    rank_m += __popc(s & ~lo);
    rank_h += __popc(live(i) & lo & ~s);
  }
  __syncthreads();
  // the lists, and the weights and positions of the slots that do not move
  const bool same_w = p.w_in == p.w_out, same_pos = p.pos_in == p.pos_out;
  for (int j0 = s0 + 4 * t; j0 < s1; j0 += U * 4 * NT) {
    float w[U][4];
    int pos[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * 4 * NT;
      if (j < min(p.keep, s1)) {
        if (!same_w) load_weights(j, w[u]);
        load_positions(j, pos[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * 4 * NT, i = (j - s0) >> 5;
      if (j >= s1) break;
      const uint32_t s = stay[i];  // s0 is a multiple of 32
      const int b = j & 31;
      // holes and movers are written again by their moves, which come later
      if (p.vec && j + 4 <= min(p.keep, s1)) {
        if (!same_w) Vec4<float>::store(w_out + j, w[u]);
        if (!(same_pos && j + 4 <= known))
          *reinterpret_cast<int4 *>(pos_out + j) = make_int4(pos[u][0], pos[u][1], pos[u][2], pos[u][3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (j + k >= s1) break;
          if (j + k < p.keep) {
            if (!same_w) w_out[j + k] = w[u][k];
            if (!(same_pos && j + k < known)) pos_out[j + k] = pos[u][k];
          } else if (!same_w || !(s >> (b + k) & 1)) {  // (in place a mover's weight is still to be read)
            w_out[j + k] = 0.f;
          }
        }
      }
      const uint32_t lo = below_keep(i), hole = live(i) & lo & ~s, mover = s & ~lo;
      for (uint32_t m = (hole | mover) >> b & 15u; m; m &= m - 1) {
        const int k = b + __ffs(m) - 1;
        const uint32_t before = (1u << k) - 1;
        if (hole >> k & 1) holes[hole0[i] + __popc(hole & before)] = j - b + k;
        else movers[equal_w[i] + __popc(mover & before)] = j - b + k;
      }
    }
  }
  if constexpr (FUSED) {
    if (C > 1) cluster_sync();
    else __syncthreads();
    const int step = moves_per_warp(p);
    for (int r0 = (part * kWarpsNT + warp) * step; r0 < moves; r0 += C * kWarpsNT * step) {
      const bool mine = r0 + lane < moves;
      move_rows(p, row, h, mine ? holes[r0 + lane] : 0, mine ? movers[r0 + lane] : 0, moves - r0);
    }
  }
  if (C > 1) cluster_sync();  // no CTA leaves while another may read its shared memory
}

constexpr int kMoveThreads = 128;

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(EvictParams p) {
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, step = moves_per_warp(p);
  const size_t pair = size_t(row) * p.num_kv_heads + h;
  const int r0 = (int(blockIdx.z) * (kMoveThreads / 32) + int(threadIdx.x >> 5)) * step;
  const int32_t *holes = p.lists + pair * 2 * size_t(p.half), *movers = holes + p.half;
  const bool mine = lane < step && r0 + lane < p.half;
  const int jt = mine ? holes[r0 + lane] : 0, jf = mine ? movers[r0 + lane] : 0;  // beside the count, not behind it
  const int count = p.moves[pair] - r0;  // (0 moves for a row that was skipped)
  if (count > 0) move_rows(p, row, h, jt, jf, count);
}

// CTAs per (sequence, kv head): enough to fill the machine (two on each of the 148 SMs), with
// at least 4096 slots each (one sequence of 2176 slots: one CTA a head 10.4 us, two 15.5: each
// digit then costs two cluster barriers), and as many as the rank keys need.
int evict_cluster(int rows, int hkv, int max_ctx) {
  int c = 1;
  while (c < kMaxCluster &&
         (max_ctx > c * kMaxSlots || ((long long)rows * hkv * c < 2 * 148 && max_ctx > 4096 * c)))
    c *= 2;
  return c;
}

size_t evict_smem(int seg) { return (size_t(seg) + 3 * (seg / 32)) * sizeof(uint32_t); }

template <int NT, bool FUSED>
cudaError_t launch_evict(const EvictParams &p, int rows, int C, cudaStream_t stream) {
  auto kern = evict_kernel<NT, FUSED>;
  const int seg = ((p.max_ctx + C - 1) / C + 31) / 32 * 32;
  static std::atomic<bool> attr_done[64];  // per device; zero-initialised (static storage)
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev].load(std::memory_order_acquire)) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(evict_smem(kMaxSlots)));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_done[dev].store(true, std::memory_order_release);  // setting twice is harmless
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(rows) * C, p.num_kv_heads);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = evict_smem(seg);
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = C;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p, C, seg);
}

cudaError_t launch_moves(const EvictParams &p, int rows, int most, cudaStream_t stream) {
  const int per_cta = kMoveThreads / 32 * 4 * (32 / p.chunks);
  const dim3 grid(rows, p.num_kv_heads, (most + per_cta - 1) / per_cta);
  evict_move_kernel<<<grid, kMoveThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

int64_t evict_workspace_bytes(int num_rows, int num_kv_heads, int max_ctx) {
  if (num_rows <= 0 || num_kv_heads <= 0 || max_ctx <= 0) return 0;
  // holes and movers (at most half of the slots each) and their number
  return int64_t(num_rows) * num_kv_heads * (2 * (max_ctx / 2 + 1) + 1) * int64_t(sizeof(int32_t));
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
      max_ctx > kMaxCluster * kMaxSlots || max_ctx > int64_t(max_blocks_per_seq) * attn::kBS || stride < max_ctx ||
      (row_table ? !ptr4(row_table) : table_rows < num_rows) || !ptr4(row_ctx) || !ptr4(row_next) ||
      (row_known && (!ptr4(row_known) || !pos_in)) || (pos_in && !ptr4(pos_in)) || !ptr4(weight_in) ||
      !ptr4(weight_out) || !ptr4(pos_out) || keep <= 0 || sinks < 0 || recent < 0 || int64_t(sinks) + recent > keep ||
      !ptr4(workspace) || workspace_bytes < evict_workspace_bytes(num_rows, num_kv_heads, max_ctx))
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
  p.chunks = head_dim * (dtype == MS_DTYPE_F32 ? 4 : 2) / 16;
  p.half = max_ctx / 2 + 1;
  p.vec = stride % 4 == 0 && ptr16(weight_in) && ptr16(weight_out) && ptr16(pos_out) && (!pos_in || ptr16(pos_in));
  p.lists = static_cast<int32_t *>(workspace);
  p.moves = p.lists + size_t(num_rows) * num_kv_heads * 2 * p.half;
  cudaError_t e = standalone_status_word(&p.status);
  if (e != cudaSuccess) return int(e);
  const int C = evict_cluster(num_rows, num_kv_heads, max_ctx);
  if ((long long)num_rows * C > 0x7fffffffLL) return int(cudaErrorInvalidValue);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int most = std::max(0, std::min(keep, max_ctx - keep));  // moves of one head
  // One launch where every warp of the cluster has at most one round of moves (one sequence, 128
  // moves a head: 13 us a call, 16 with a second launch, which costs the host more than the GPU;
  // 64 sequences with up to 512 moves: 124 us of GPU time in one launch, 43 in two).
  if ((long long)most <= C * (512LL / 32) * 4 * (32 / p.chunks)) return int(launch_evict<512, true>(p, num_rows, C, st));
  // small CTAs, four to an SM, where there are enough of them to fill it that way (64 sequences:
  // 43 us, CTAs of 512 46 us)
  const bool many = (long long)num_rows * num_kv_heads * C >= 2 * 148;
  e = many ? launch_evict<256, false>(p, num_rows, C, st) : launch_evict<512, false>(p, num_rows, C, st);
  if (e == cudaSuccess) e = launch_moves(p, num_rows, most, st);
  return int(e);
}
