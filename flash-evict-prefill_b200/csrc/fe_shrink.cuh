// Eviction from a cache back to its budget, in place.
//
// A row (b, h) of n > budget tokens keeps the `budget` largest by
//   (position > newest - recent) first, then mass (NaN above every number),
//   then the lower slot,
// newest being the row's largest position.  The kept tokens below slot
// `budget` stay where they are; the i-th evicted slot below it (a hole) takes
// the i-th kept token at or above it (a mover).  So sources all lie at or above
// the budget and destinations below it: nothing that is still to be read is
// overwritten, and only min(evicted, budget) rows at most move -- one row after
// a decode step that is one token over, where keeping the slots in order would
// move nearly all of them.  A cached key carries its rotary position, so the
// order of the slots means nothing to the attention.
//
// One cluster of CTAs per row, every warp a contiguous stretch of slots.  Keys
// are order-preserving integers; the budget-th largest is found by four 8-bit
// radix passes whose histograms are summed over distributed shared memory.
// Holes and movers are then numbered by ballots in slot order, listed, and
// copied by all warps of the cluster.
#pragma once

#include <cooperative_groups.h>

#include "fe_decode.cuh"
#include "fe_select.cuh"

namespace fe {

struct ShrinkParams {
  uint8_t* k;
  int64_t k_sb, k_sh, k_st;  // bytes
  uint8_t* v;
  int64_t v_sb, v_sh, v_st;
  const float* mass_in;
  const float* norms_in;  // or null
  const int32_t* pos_in;
  const int32_t* len_in;
  float* mass_out;
  float* norms_out;
  int32_t* pos_out;
  int32_t* len_out;
  int32_t* holes;   // workspace [rows][list]
  int32_t* movers;  // workspace [rows][list]
  int64_t list;
  int Hkv, capacity, budget, recent, row_bytes;
  int copy;  // the outputs are other buffers than the inputs
};

constexpr int SHRINK_THREADS = 512;
constexpr int SHRINK_WARPS = SHRINK_THREADS / 32;
constexpr int SHRINK_SMEM_KEYS = 49152;  // keys a CTA keeps in shared memory

// Copies row `src` to row `dst` of the cache's K and V by one warp.
__device__ __forceinline__ void shrink_move(uint8_t* kb, int64_t k_st, uint8_t* vb, int64_t v_st, int row_bytes, int src,
                                            int dst, int lane) {
  const uint8_t* ks = kb + src * k_st;
  const uint8_t* vs = vb + src * v_st;
  uint8_t* kd = kb + dst * k_st;
  uint8_t* vd = vb + dst * v_st;
  const int vec = row_bytes / 16;  // rows start on 16 bytes
  for (int c = lane; c < 2 * vec; c += 32) {
    const bool is_v = c >= vec;
    const int o = (is_v ? c - vec : c) * 16;
    *reinterpret_cast<uint4*>((is_v ? vd : kd) + o) = *reinterpret_cast<const uint4*>((is_v ? vs : ks) + o);
  }
  for (int o = vec * 16 + lane * 2; o < row_bytes; o += 64) {
    *reinterpret_cast<uint16_t*>(kd + o) = *reinterpret_cast<const uint16_t*>(ks + o);
    *reinterpret_cast<uint16_t*>(vd + o) = *reinterpret_cast<const uint16_t*>(vs + o);
  }
}

template <bool SMEM_KEYS>
__global__ void __launch_bounds__(SHRINK_THREADS) fe_shrink_kernel(const __grid_constant__ ShrinkParams p) {
  extern __shared__ uint32_t skeys[];
  __shared__ uint32_t hist[2][256];
  __shared__ int warp_count[3][SHRINK_WARPS];  // ties, holes, movers of each warp
  __shared__ int found[2];
  __shared__ int smax[SHRINK_WARPS], cta_max;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), size = static_cast<int>(cluster.num_blocks());
  const int row = static_cast<int>(blockIdx.x) / size;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = cache_length(p.len_in, row, p.capacity);
  const int64_t base = static_cast<int64_t>(row) * p.capacity;
  const float* mass = p.mass_in + base;
  const int32_t* pos = p.pos_in + base;

  if (n <= p.budget) {
    if (p.copy) {
      for (int i = rank * SHRINK_THREADS + tid; i < n; i += size * SHRINK_THREADS) {
        p.mass_out[base + i] = mass[i];
        p.pos_out[base + i] = pos[i];
        if (p.norms_in != nullptr) p.norms_out[base + i] = p.norms_in[base + i];
      }
    }
    cluster.sync();  // every CTA has read the length
    if (rank == 0 && tid == 0) p.len_out[row] = n;
    return;
  }

  // This warp's slots: [w0, w1).
  const int wlen = ((n + size * SHRINK_WARPS - 1) / (size * SHRINK_WARPS) + 31) & ~31;
  const int w0 = min(n, (rank * SHRINK_WARPS + warp) * wlen), w1 = min(n, w0 + wlen);

  int first_reserved = 0;  // positions from here on are reserved (recent > 0)
  if (p.recent > 0) {
    int newest = -0x7fffffff - 1;
    for (int i = w0 + lane; i < w1; i += 32) newest = max(newest, pos[i]);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) smax[warp] = newest;
    __syncthreads();
    if (tid == 0) {
      int m = smax[0];
      for (int w = 1; w < SHRINK_WARPS; ++w) m = max(m, smax[w]);
      cta_max = m;
    }
    cluster.sync();
    newest = cta_max;
    for (int r = 0; r < size; ++r) newest = max(newest, *cluster.map_shared_rank(&cta_max, r));
    first_reserved = static_cast<int>(max(static_cast<int64_t>(newest) - p.recent + 1, static_cast<int64_t>(-0x80000000LL)));
  }
  auto make_key = [&](int i) -> uint32_t {
    if (p.recent > 0 && pos[i] >= first_reserved) return 0xFFFFFFFFu;
    // NaN below the reserved tokens, above +inf
    return min(order_key(mass[i]), 0xFFFFFFFEu);
  };
  uint32_t* wkeys = skeys + warp * wlen;
  auto key_at = [&](int i) -> uint32_t { return SMEM_KEYS ? wkeys[i - w0] : make_key(i); };
  if (SMEM_KEYS)
    for (int i = w0 + lane; i < w1; i += 32) wkeys[i - w0] = make_key(i);

  // ---- the budget-th largest key
  uint32_t prefix = 0u;
  int need = p.budget, ties = 0;
  for (int i = tid; i < 512; i += SHRINK_THREADS) hist[i >> 8][i & 255] = 0u;
  __syncthreads();
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    uint32_t* hh = hist[pass & 1];
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t key = i < w1 ? key_at(i) : 0u;
      const bool in = i < w1 && (pass == 0 || (key >> (shift + 8)) == (prefix >> (shift + 8)));
      const uint32_t digit = in ? (key >> shift) & 255u : 256u;
      // The keys crowd into few digits: add once per distinct digit of the warp.
      const uint32_t same = __match_any_sync(0xffffffffu, digit);
      if (in && (__ffs(same) - 1) == lane) atomicAdd(&hh[digit], static_cast<uint32_t>(__popc(same)));
    }
    cluster.sync();
    // Every CTA sums the clusters' histograms and finds the digit (warp 0).
    if (warp == 0) {
      uint32_t cnt[8];
      uint32_t mine = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        cnt[u] = 0;
        for (int r = 0; r < size; ++r) cnt[u] += *cluster.map_shared_rank(&hh[lane * 8 + u], r);
        mine += cnt[u];
      }
      uint32_t above = mine;  // inclusive suffix sum over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_down_sync(0xffffffffu, above, o);
        if (lane + o < 32) above += x;
      }
      uint32_t upper = above - mine;  // keys in higher lanes' digits
#pragma unroll
      for (int u = 7; u >= 0; --u) {
        if (upper < static_cast<uint32_t>(need) && upper + cnt[u] >= static_cast<uint32_t>(need)) {
          found[0] = lane * 8 + u;
          found[1] = static_cast<int>(upper);
          warp_count[0][0] = static_cast<int>(cnt[u]);
        }
        upper += cnt[u];
      }
    }
    // The other histogram is free: every CTA is past reading it.
    if (warp > 0 && pass < 3)
      for (int i = tid - 32; i < 256; i += SHRINK_THREADS - 32) hist[(pass + 1) & 1][i] = 0u;
    __syncthreads();
    prefix |= static_cast<uint32_t>(found[0]) << shift;
    need -= found[1];
    ties = warp_count[0][0];
    __syncthreads();
  }
  const uint32_t threshold = prefix;
  const int keep_ties = need;  // of `ties` keys equal to it, the first ones stay

  auto prefix_of = [&](int which) -> int {
    // Sum of warp_count[which] over the warps before this one, in the cluster.
    int s = 0;
    for (int i = lane; i < rank * SHRINK_WARPS + warp; i += 32)
      s += *cluster.map_shared_rank(&warp_count[which][i % SHRINK_WARPS], i / SHRINK_WARPS);
    return __reduce_add_sync(0xffffffffu, s);
  };
  int tie_base = 0;
  if (ties > keep_ties) {
    int c = 0;
    for (int i = w0 + lane; i < w1; i += 32) c += key_at(i) == threshold ? 1 : 0;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) warp_count[0][warp] = c;
    cluster.sync();
    tie_base = prefix_of(0);
  }
  // Calls f(slot, valid, kept) for the warp's slots, 32 at a time in order.
  auto sweep = [&](auto f) {
    int seen = tie_base;
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      const bool valid = i < w1;
      const uint32_t key = valid ? key_at(i) : 0u;
      bool keep = valid && key >= threshold;
      if (ties > keep_ties) {
        const bool tie = valid && key == threshold;
        const uint32_t bal = __ballot_sync(0xffffffffu, tie);
        if (tie) keep = seen + __popc(bal & ((1u << lane) - 1u)) < keep_ties;
        seen += __popc(bal);
      }
      f(i, valid, keep);
    }
  };
  int nh = 0, nm = 0;
  sweep([&](int i, bool valid, bool keep) {
    nh += __popc(__ballot_sync(0xffffffffu, valid && !keep && i < p.budget));
    nm += __popc(__ballot_sync(0xffffffffu, keep && i >= p.budget));
  });
  if (lane == 0) {
    warp_count[1][warp] = nh;
    warp_count[2][warp] = nm;
  }
  cluster.sync();
  int hole = prefix_of(1), mover = prefix_of(2);
  int32_t* holes = p.holes + static_cast<int64_t>(row) * p.list;
  int32_t* movers = p.movers + static_cast<int64_t>(row) * p.list;
  sweep([&](int i, bool valid, bool keep) {
    const bool is_hole = valid && !keep && i < p.budget, is_mover = keep && i >= p.budget;
    const uint32_t bh = __ballot_sync(0xffffffffu, is_hole), bm = __ballot_sync(0xffffffffu, is_mover);
    const uint32_t below = (1u << lane) - 1u;
    if (is_hole) holes[hole + __popc(bh & below)] = i;
    if (is_mover) movers[mover + __popc(bm & below)] = i;
    hole += __popc(bh);
    mover += __popc(bm);
    if (p.copy && keep && i < p.budget) {
      p.mass_out[base + i] = mass[i];
      p.pos_out[base + i] = pos[i];
      if (p.norms_in != nullptr) p.norms_out[base + i] = p.norms_in[base + i];
    }
  });
  int moves = 0;
  for (int i = lane; i < size * SHRINK_WARPS; i += 32)
    moves += *cluster.map_shared_rank(&warp_count[1][i % SHRINK_WARPS], i / SHRINK_WARPS);
  moves = __reduce_add_sync(0xffffffffu, moves);
  __threadfence();
  cluster.sync();  // the lists are complete, and nobody reads a neighbour's shared memory any more
  if (rank == 0 && tid == 0) p.len_out[row] = p.budget;
  const int b = row / p.Hkv, h = row - b * p.Hkv;
  uint8_t* kb = p.k + b * p.k_sb + h * p.k_sh;
  uint8_t* vb = p.v + b * p.v_sb + h * p.v_sh;
  for (int i = rank * SHRINK_WARPS + warp; i < moves; i += size * SHRINK_WARPS) {
    const int dst = __ldcg(holes + i), src = __ldcg(movers + i);
    shrink_move(kb, p.k_st, vb, p.v_st, p.row_bytes, src, dst, lane);
    if (lane == 0) {
      p.mass_out[base + dst] = mass[src];
      p.pos_out[base + dst] = pos[src];
      if (p.norms_in != nullptr) p.norms_out[base + dst] = p.norms_in[base + src];
    }
  }
}

}  // namespace fe
