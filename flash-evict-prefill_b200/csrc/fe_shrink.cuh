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
// One cluster of CTAs per row, every warp a contiguous stretch of slots whose
// order-preserving integer keys stay in shared memory (in registers the walks
// over them have to be unrolled, and fetching that code once took longer than
// running it: 46 us instead of 40 for eight rows of 128K when that was all that
// differed; the whole takes 28 now).  The budget-th largest key is
// found by narrowing the range of the keys 1024-fold a pass (bins of a power of
// two from the row's smallest key, so keys that share their top bits spread over
// the bins all the same), histograms summed over distributed shared memory,
// ending as soon as a bin's end coincides with the budget (one or two passes for
// a row of a few thousand).  Holes and movers are numbered by ballots in slot order,
// listed, and copied by all warps of the cluster, eight rows a warp in flight.
// Where that leaves some SM much more to copy than others (few rows, rows with
// very different numbers of moves), a second launch splits all rows' moves evenly.
// Few rows are bound by the chain of cluster barriers, large batches by the moved
// bytes.
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
  int32_t* counts;  // workspace [rows]: moves of each row, or null: moved by this launch
  int64_t list;
  int rows, Hkv, capacity, budget, recent, row_bytes;
  int copy;  // the outputs are other buffers than the inputs
  int hold_positions;  // shared memory holds the positions, too
};

constexpr int SHRINK_THREADS = 1024;
constexpr int SHRINK_WARPS = SHRINK_THREADS / 32;
static_assert(SHRINK_WARPS == 32, "scans give a lane to every warp");
constexpr int SHRINK_MAX_CLUSTER = 8;
// Keys a CTA holds.  (Clusters of 16 fit fewer than one to a GPC and ran eight
// rows of 128K one after another.)
constexpr int SHRINK_SMEM_KEYS = 49152;
constexpr int SHRINK_BINS = 1024;  // bins of a pass, one a thread
constexpr int SHRINK_LIST = 1024;  // moves listed in shared memory (one CTA a row)

// Copies rows src[u] to rows dst[u], u < count <= U, of a cache's K and V by one
// warp: all loads before the first store.
template <int U>
__device__ __forceinline__ void shrink_move(const ShrinkParams& p, uint8_t* kb, uint8_t* vb, const int* src,
                                            const int* dst, int count, int lane) {
  const int vec = p.row_bytes / 16;  // rows start on 16 bytes
  for (int c = lane; c < 2 * vec; c += 32) {
    const bool is_v = c >= vec;
    uint8_t* at = (is_v ? vb : kb) + (is_v ? c - vec : c) * 16;
    const int64_t st = is_v ? p.v_st : p.k_st;
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < count) x[u] = *reinterpret_cast<const uint4*>(at + src[u] * st);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < count) *reinterpret_cast<uint4*>(at + dst[u] * st) = x[u];
  }
  for (int o = vec * 16 + lane * 2; o < p.row_bytes; o += 64)
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < count) {
        *reinterpret_cast<uint16_t*>(kb + dst[u] * p.k_st + o) = *reinterpret_cast<const uint16_t*>(kb + src[u] * p.k_st + o);
        *reinterpret_cast<uint16_t*>(vb + dst[u] * p.v_st + o) = *reinterpret_cast<const uint16_t*>(vb + src[u] * p.v_st + o);
      }
}

// Moves [i0, end) of a row, eight consecutive ones a warp at a time (`step`
// apart), lane u < 8 knowing the u-th; the next ones are looked up, and the
// bookkeeping read, while the rows are on their way.
template <typename Look>
__device__ __forceinline__ void shrink_moves(const ShrinkParams& p, int row, int i0, int end, int step, int lane, Look look) {
  constexpr int U = 8;
  const int b = row / p.Hkv, h = row - b * p.Hkv;
  const int64_t base = static_cast<int64_t>(row) * p.capacity;
  uint8_t* kb = p.k + b * p.k_sb + h * p.k_sh;
  uint8_t* vb = p.v + b * p.v_sb + h * p.v_sh;
  auto mine_of = [&](int i) { return lane < U && i + lane < end ? look(i + lane) : make_int2(0, 0); };
  int2 mine = mine_of(i0);  // {hole, mover}
  for (; i0 < end; i0 += step) {
    const int count = min(U, end - i0);
    const int2 next = mine_of(i0 + step);
    float m = 0.f, z = 0.f;
    int at = 0;
    if (lane < count) {
      m = p.mass_in[base + mine.y];
      at = p.pos_in[base + mine.y];
      if (p.norms_in != nullptr) z = p.norms_in[base + mine.y];
    }
    int src[U], dst[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      dst[u] = __shfl_sync(0xffffffffu, mine.x, u);
      src[u] = __shfl_sync(0xffffffffu, mine.y, u);
    }
    shrink_move<U>(p, kb, vb, src, dst, count, lane);
    if (lane < count) {
      p.mass_out[base + mine.x] = m;
      p.pos_out[base + mine.x] = at;
      if (p.norms_in != nullptr) p.norms_out[base + mine.x] = z;
    }
    mine = next;
  }
}

// HELD: the keys of a CTA's slots fit its shared memory; otherwise (longer rows)
// they are made again from the weights on every walk.
template <bool HELD>
__global__ void __launch_bounds__(SHRINK_THREADS, 1) fe_shrink_kernel(const __grid_constant__ ShrinkParams p) {
  extern __shared__ uint32_t skeys[];
  __shared__ uint32_t hist[2][SHRINK_BINS + 1];  // the last bin counts the reserved tokens
  __shared__ __align__(16) uint32_t sums[3][SHRINK_BINS + 4];  // the cluster's histogram of a pass, each CTA some bins
  __shared__ int2 warp_count[2][SHRINK_WARPS];  // ties; holes and movers of each warp
  __shared__ int2 cta_count[2];
  __shared__ int found[3];
  __shared__ int s_new[SHRINK_WARPS], cta_new;
  __shared__ uint32_t s_lo[SHRINK_WARPS], s_hi[SHRINK_WARPS], cta_lo, cta_hi;
  __shared__ int2 slist[SHRINK_LIST];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), size = static_cast<int>(cluster.num_blocks());
  const int row = static_cast<int>(blockIdx.x) / size;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int n = cache_length(p.len_in, row, p.capacity);
  const int64_t base = static_cast<int64_t>(row) * p.capacity;
  const float* mass = p.mass_in + base;
  const int32_t* pos = p.pos_in + base;
  auto sync = [&] {
    if (size > 1) cluster.sync();
    else __syncthreads();
  };

  if (n <= p.budget) {
    if (p.copy) {
      for (int i = rank * SHRINK_THREADS + tid; i < n; i += size * SHRINK_THREADS) {
        p.mass_out[base + i] = mass[i];
        p.pos_out[base + i] = pos[i];
        if (p.norms_in != nullptr) p.norms_out[base + i] = p.norms_in[base + i];
      }
    }
    sync();  // every CTA has read the length
    if (rank == 0 && tid == 0) {
      p.len_out[row] = n;
      if (p.counts != nullptr) p.counts[row] = 0;
    }
    return;
  }

  // This warp's slots: [w0, w1), lane l holding w0 + l, w0 + l + 32, ...
  const int wlen = ((n + size * SHRINK_WARPS - 1) / (size * SHRINK_WARPS) + 31) & ~31;
  const int w0 = min(n, (rank * SHRINK_WARPS + warp) * wlen), w1 = min(n, w0 + wlen);
  const int steps = (w1 - w0 + 31) >> 5;

  uint32_t* wkeys = skeys + warp * wlen;
  int* wpos = reinterpret_cast<int*>(skeys + SHRINK_WARPS * wlen) + warp * wlen;  // p.hold_positions
  int first_reserved = 0;  // positions from here on are reserved (recent > 0)
  uint32_t lo = 0xFFFFFFFFu, hi = 0u;  // range of the row's weights
  auto mass_key = [&](float m) -> uint32_t { return min(order_key(m), 0xFFFFFFFEu); };  // NaN above +inf, below the reserved
  auto as_key = [&](uint32_t k, int at) -> uint32_t { return p.recent > 0 && at >= first_reserved ? 0xFFFFFFFFu : k; };
  {
    int newest = -0x7fffffff - 1;
    // Loads of eight slots at a time, past the end from the last slot.
    for (int j0 = 0; j0 < steps; j0 += 8) {
      float m[8], z[8];
      int at[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = min(w0 + (j0 + u) * 32 + lane, n - 1);
        m[u] = mass[i];
        at[u] = p.recent > 0 || p.copy ? pos[i] : 0;
        if (p.copy && p.norms_in != nullptr) z[u] = p.norms_in[base + i];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = w0 + (j0 + u) * 32 + lane;
        const uint32_t k = mass_key(m[u]);
        lo = min(lo, k);
        hi = max(hi, k);
        newest = max(newest, at[u]);
        if (HELD && j0 + u < steps) {
          wkeys[(j0 + u) * 32 + lane] = i < w1 ? k : 0u;  // past the row's end: below every weight
          if (p.hold_positions) wpos[(j0 + u) * 32 + lane] = at[u];
        }
        if (p.copy && i < min(w1, p.budget)) {
          // The evicted ones are overwritten after a barrier.
          p.mass_out[base + i] = m[u];
          p.pos_out[base + i] = at[u];
          if (p.norms_in != nullptr) p.norms_out[base + i] = z[u];
        }
      }
    }
    for (int i = tid; i <= SHRINK_BINS; i += SHRINK_THREADS) {
      hist[0][i] = hist[1][i] = 0u;
      sums[0][i] = sums[1][i] = sums[2][i] = 0u;
    }
    newest = __reduce_max_sync(0xffffffffu, newest);
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      s_new[warp] = newest;
      s_lo[warp] = lo;
      s_hi[warp] = hi;
    }
    __syncthreads();
    newest = __reduce_max_sync(0xffffffffu, s_new[lane % SHRINK_WARPS]);
    lo = __reduce_min_sync(0xffffffffu, s_lo[lane % SHRINK_WARPS]);
    hi = __reduce_max_sync(0xffffffffu, s_hi[lane % SHRINK_WARPS]);
    if (size > 1) {
      if (tid == 0) {
        cta_new = newest;
        cta_lo = lo;
        cta_hi = hi;
      }
      cluster.sync();
      const int r = lane < size ? lane : 0;
      newest = __reduce_max_sync(0xffffffffu, *cluster.map_shared_rank(&cta_new, r));
      lo = __reduce_min_sync(0xffffffffu, *cluster.map_shared_rank(&cta_lo, r));
      hi = __reduce_max_sync(0xffffffffu, *cluster.map_shared_rank(&cta_hi, r));
    }
    first_reserved =
        static_cast<int>(max(static_cast<int64_t>(newest) - p.recent + 1, static_cast<int64_t>(-0x80000000LL)));
    if (HELD && p.recent > 0 && p.hold_positions) {
#pragma unroll 4
      for (int j = 0; j < steps; ++j) {
        const int i = j * 32 + lane;
        if (w0 + i < w1 && wpos[i] >= first_reserved) wkeys[i] = 0xFFFFFFFFu;
      }
    } else if (HELD && p.recent > 0) {
      for (int j0 = 0; j0 < steps; j0 += 8) {
        int at[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) at[u] = pos[min(w0 + (j0 + u) * 32 + lane, n - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (at[u] >= first_reserved && w0 + (j0 + u) * 32 + lane < w1) wkeys[(j0 + u) * 32 + lane] = 0xFFFFFFFFu;
      }
    }
    __syncwarp();
  }
  // Calls f(slot, key) for the warp's slots, 32 at a time in order; the key is 0,
  // below every weight's, past the row's end.
  auto walk = [&](auto f) {
#pragma unroll 4
    for (int j = 0; j < steps; ++j) {
      const int i = w0 + j * 32 + lane;
      uint32_t k = 0u;
      if (HELD) k = wkeys[j * 32 + lane];
      else if (i < w1) k = as_key(mass_key(mass[i]), p.recent > 0 ? pos[i] : 0);
      f(i, k);
    }
  };

  // ---- the budget-th largest key
  const int owner = tid * size / SHRINK_BINS;  // CTA that gathers this thread's bin
  // Candidates are the keys in [threshold, threshold + span]; bins of 2^shift of
  // them.  (A reserved token's key is above any such range.)
  uint32_t threshold = lo, span = hi - lo;
  int need = p.budget, ties = 0;
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {  // 32 bits, 10 a pass
    const int shift = max(22 - __clz(span), 0);
    uint32_t* hh = hist[pass & 1];
    int reserved_here = 0;
    walk([&](int, uint32_t k) {
      const uint32_t d = k - threshold;
      const bool in = d <= span;
      // Lane 0's bin once for all lanes that share it (weights of exactly zero
      // can be most of a row), the others one by one.
      const uint32_t bin = in ? d >> shift : SHRINK_BINS;
      const uint32_t first_bin = __shfl_sync(0xffffffffu, bin, 0);
      const uint32_t same = __ballot_sync(0xffffffffu, bin == first_bin);
      if (in) {
        if (bin != first_bin) atomicAdd(&hh[bin], 1u);
        else if (lane == 0) atomicAdd(&hh[bin], static_cast<uint32_t>(__popc(same)));
      }
      reserved_here += k == 0xFFFFFFFFu ? 1 : 0;
    });
    if (pass == 0 && p.recent > 0) {
      reserved_here = __reduce_add_sync(0xffffffffu, reserved_here);
      if (lane == 0 && reserved_here > 0) atomicAdd(&hh[SHRINK_BINS], static_cast<uint32_t>(reserved_here));
    }
    // The cluster's histogram gathers in three buffers: one is read, the next is
    // added to, the one after is zeroed, between two cluster barriers.
    if (size > 1) {
      __syncthreads();
      // Every CTA gathers its share of the bins.
      if (hh[tid] != 0u) atomicAdd(cluster.map_shared_rank(&sums[pass % 3][tid], owner), hh[tid]);
      if (tid == 0 && hh[SHRINK_BINS] != 0u) atomicAdd(cluster.map_shared_rank(&sums[pass % 3][SHRINK_BINS], 0), hh[SHRINK_BINS]);
    }
    sync();
    const uint32_t cnt = size > 1 ? *cluster.map_shared_rank(&sums[pass % 3][tid], owner) : hh[tid];
    const uint32_t reserved =  // (only the first pass counts reserved tokens)
        size > 1 ? *cluster.map_shared_rank(&sums[pass % 3][SHRINK_BINS], 0) : hh[SHRINK_BINS];
    for (int i = tid; i <= SHRINK_BINS; i += SHRINK_THREADS) {
      hist[(pass + 1) & 1][i] = 0u;
      sums[(pass + 2) % 3][i] = 0u;
    }
    // The bin in which the count from above reaches `need`: a suffix sum.
    uint32_t above = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_down_sync(0xffffffffu, above, o);
      if (lane + o < 32) above += x;
    }
    if (lane == 0) s_lo[warp] = above;
    __syncthreads();
    const uint32_t higher = __reduce_add_sync(0xffffffffu, lane > warp ? s_lo[lane] : 0u);
    const uint32_t upper = reserved + higher + above - cnt;  // keys above this bin
    if (upper < static_cast<uint32_t>(need) && upper + cnt >= static_cast<uint32_t>(need)) {
      found[0] = tid;
      found[1] = static_cast<int>(upper);
      found[2] = static_cast<int>(cnt);
    }
    if (tid == 0 && reserved >= static_cast<uint32_t>(need)) {
      found[0] = SHRINK_BINS;
      found[1] = 0;
      found[2] = static_cast<int>(reserved);
    }
    __syncthreads();
    const int bin = found[0];
    need -= found[1];
    ties = found[2];
    if (bin == SHRINK_BINS) {
      threshold = 0xFFFFFFFFu;
      break;
    }
    threshold += static_cast<uint32_t>(bin) << shift;
    // Done when all keys of this bin stay, or it holds one key.
    if (ties == need || shift == 0) break;
    span = (1u << shift) - 1u;
    __syncthreads();
  }
  const int keep_ties = need;  // of `ties` keys equal to it, the first ones stay
  const bool split_ties = ties > keep_ties;

  // Sums of a pair of counts over the warps before this one, in the whole
  // cluster; the cluster's totals in *total.
  auto scan = [&](int which, int2 mine, int2* total) -> int2 {
    if (lane == 0) warp_count[which][warp] = mine;
    __syncthreads();
    const int2 v = warp_count[which][lane];
    int2 before = make_int2(__reduce_add_sync(0xffffffffu, lane < warp ? v.x : 0),
                            __reduce_add_sync(0xffffffffu, lane < warp ? v.y : 0));
    int2 all = make_int2(__reduce_add_sync(0xffffffffu, v.x), __reduce_add_sync(0xffffffffu, v.y));
    if (size > 1) {
      if (tid == 0) cta_count[which] = all;
      cluster.sync();
      int2 c = make_int2(0, 0);
      if (lane < size) c = *cluster.map_shared_rank(&cta_count[which], lane);
      before.x += __reduce_add_sync(0xffffffffu, lane < rank ? c.x : 0);
      before.y += __reduce_add_sync(0xffffffffu, lane < rank ? c.y : 0);
      all = make_int2(__reduce_add_sync(0xffffffffu, c.x), __reduce_add_sync(0xffffffffu, c.y));
    }
    *total = all;
    return before;
  };
  const uint32_t below = (1u << lane) - 1u;
  int tie_base = 0;
  int2 total;
  if (split_ties) {
    int c = 0;
    walk([&](int, uint32_t k) { c += k == threshold ? 1 : 0; });
    c = __reduce_add_sync(0xffffffffu, c);
    tie_base = scan(0, make_int2(c, 0), &total).x;
  }
  // Calls f(slot, kept) in order.
  auto sweep = [&](auto f) {
    int seen = tie_base;
    walk([&](int i, uint32_t k) {
      bool keep = k >= threshold;
      if (split_ties) {
        const bool tie = k == threshold;
        const uint32_t bal = __ballot_sync(0xffffffffu, tie);
        if (tie) keep = seen + __popc(bal & below) < keep_ties;
        seen += __popc(bal);
      }
      f(i, keep);
    });
  };
  // Slots past the row's end are above the budget and not kept: neither.
  int nh = 0, nm = 0;
  sweep([&](int i, bool keep) {
    nh += !keep && i < p.budget ? 1 : 0;
    nm += keep && i >= p.budget ? 1 : 0;
  });
  nh = __reduce_add_sync(0xffffffffu, nh);
  nm = __reduce_add_sync(0xffffffffu, nm);
  const int2 start = scan(1, make_int2(nh, nm), &total);
  int hole = start.x, mover = start.y;
  const int moves = total.x;  // as many holes as movers
  // One CTA with few moves lists them in shared memory.
  const bool local = size == 1 && moves <= SHRINK_LIST && p.counts == nullptr;
  int32_t* holes = p.holes + static_cast<int64_t>(row) * p.list;
  int32_t* movers = p.movers + static_cast<int64_t>(row) * p.list;
  sweep([&](int i, bool keep) {
    const bool is_hole = !keep && i < p.budget, is_mover = keep && i >= p.budget;
    const uint32_t bh = __ballot_sync(0xffffffffu, is_hole), bm = __ballot_sync(0xffffffffu, is_mover);
    if (is_hole) {
      if (local) slist[hole + __popc(bh & below)].x = i;
      else holes[hole + __popc(bh & below)] = i;
    }
    if (is_mover) {
      if (local) slist[mover + __popc(bm & below)].y = i;
      else movers[mover + __popc(bm & below)] = i;
    }
    hole += __popc(bh);
    mover += __popc(bm);
  });
  if (!local) __threadfence();
  sync();  // the lists are complete, and nobody reads a neighbour's shared memory any more
  if (rank == 0 && tid == 0) p.len_out[row] = p.budget;
  if (p.counts != nullptr) {
    if (rank == 0 && tid == 0) p.counts[row] = moves;
    return;
  }
  shrink_moves(p, row, (rank * SHRINK_WARPS + warp) * 8, moves, size * SHRINK_WARPS * 8, lane, [&](int i) {
    return local ? slist[i] : make_int2(__ldcg(holes + i), __ldcg(movers + i));
  });
}

constexpr int MOVE_THREADS = 512;

// The rows' moves laid end to end, an equal run for every CTA.
__global__ void __launch_bounds__(MOVE_THREADS, 1) fe_shrink_move_kernel(const __grid_constant__ ShrinkParams p) {
  __shared__ int sums[MOVE_THREADS / 32];
  __shared__ int found[2];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_thread = (p.rows + MOVE_THREADS - 1) / MOVE_THREADS;
  const int first = min(p.rows, static_cast<int>(threadIdx.x) * per_thread), last = min(p.rows, first + per_thread);
  int mine = 0;
  for (int i = first; i < last; ++i) mine += __ldcg(p.counts + i);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int start = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < MOVE_THREADS / 32; ++w) {
    start += w < warp ? sums[w] : 0;
    total += sums[w];
  }
  // Runs of whole groups of eight, so that a group of a row is not shared.
  const int per = ((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x) + 7) & ~7;
  const int lo = min(total, static_cast<int>(blockIdx.x) * per), hi = min(total, lo + per);
  for (int i = first; i < last; ++i) {
    const int n = __ldcg(p.counts + i);
    if (lo < hi && start <= lo && lo < start + n) {
      found[0] = i;
      found[1] = start;
    }
    start += n;
  }
  __syncthreads();
  if (lo >= hi) return;
  int row = found[0], begin = found[1];  // first move of `row` in the whole
  while (begin < hi) {
    const int n = __ldcg(p.counts + row);
    const int32_t* holes = p.holes + static_cast<int64_t>(row) * p.list;
    const int32_t* movers = p.movers + static_cast<int64_t>(row) * p.list;
    shrink_moves(p, row, max(lo - begin, 0) + warp * 8, min(hi - begin, n), MOVE_THREADS / 32 * 8, lane,
                 [&](int i) { return make_int2(__ldcg(holes + i), __ldcg(movers + i)); });
    begin += n;
    ++row;
  }
}

}  // namespace fe
