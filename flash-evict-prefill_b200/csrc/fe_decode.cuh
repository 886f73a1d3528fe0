// What the decode kernels share: the cache as the kernels see it and the even
// split of all (row, key tile) work over the CTAs of one launch.
//
// A cache row (b, hkv) uses its first lengths[b*Hkv + hkv] slots.  The lengths
// live on the device and change from step to step, so the host sizes a launch
// by the capacity alone and the CTAs divide the real work among themselves:
// the rows' key tiles, laid end to end, are cut into equal runs.  A run may
// begin and end inside a row (a long row is shared by many CTAs, a batch of
// short rows by few), which keeps every SM busy whatever the lengths are.
#pragma once

#include "fe_ptx.cuh"

namespace fe {

constexpr int DEC_TILE = 128;  // keys per tile

__device__ __forceinline__ int cache_length(const int32_t* lengths, int bh, int capacity) {
  return min(max(lengths[bh], 0), capacity);
}

// One contiguous run of a row's tiles: tiles [j0, j1) of `tiles` for row tile mt.
struct DecSegment {
  int bh, mt, j0, j1, tiles, len;
};

// Walks the segments of one CTA's run.  A row bh has MT * (tiles(bh) + extra)
// units: MT row tiles of queries, each over all of the row's key tiles (the
// cache's and one of drafted tokens) and `extra` units of no work, which stand
// for what a run spends on beginning and ending a row.
struct DecWalk {
  const int32_t* lengths;
  int capacity, mts, extra, bh, unit, left;
  __device__ __forceinline__ bool next(DecSegment& s) {
    while (left > 0) {
      s.bh = bh;
      s.len = cache_length(lengths, bh, capacity);
      s.tiles = (s.len + DEC_TILE - 1) / DEC_TILE + 1;
      const int span = s.tiles + extra;
      s.mt = unit / span;
      s.j0 = unit - s.mt * span;
      const int n = min(left, span - s.j0);
      s.j1 = min(s.j0 + n, s.tiles);
      left -= n;
      unit += n;
      if (unit == mts * span) {
        unit = 0;
        ++bh;
      }
      if (s.j1 > s.j0) return true;
    }
    return false;
  }
};

constexpr int DEC_SCRATCH_INTS = 36;

// Units that stand for a row's beginning and end in a launch of `total` key
// tiles: with few tiles a run they would only spread the work over fewer SMs.
__device__ __forceinline__ int dec_extra(int total, int nctas, int extra) { return total >= 4 * nctas ? extra : 0; }

// The layout of the units: first unit of the rows and their total.
struct DecLayout {
  int total, per, extra;  // units, units a run, extra units a row tile
};

// Sums the rows' units; every thread gets the layout and the first unit of its
// own rows [first, last).  All THREADS threads call it (one block barrier;
// scratch is free again after the next one).
template <int THREADS>
__device__ __forceinline__ DecLayout dec_layout(const int32_t* lengths, int nbh, int capacity, int mts, int extra, int nctas,
                                                int* scratch, int& first, int& last, int& start) {
  constexpr int WARPS = THREADS / 32;
  static_assert(WARPS <= 32 && THREADS % 32 == 0, "one warp scans the warps' sums");
  const int per_thread = (nbh + THREADS - 1) / THREADS;
  first = min(nbh, static_cast<int>(threadIdx.x) * per_thread);
  last = min(nbh, first + per_thread);
  int mine = 0;
  for (int i = first; i < last; ++i)
    mine += mts * ((cache_length(lengths, i, capacity) + DEC_TILE - 1) / DEC_TILE + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int v = scratch[w];
    before += w < warp ? v : 0;
    total += v;
  }
  DecLayout d;
  d.extra = dec_extra(total, nctas, extra);
  d.total = total + nbh * mts * d.extra;
  d.per = (d.total + nctas - 1) / nctas;
  start = before + incl - mine + first * mts * d.extra;
  return d;
}

// Where this CTA's run starts.  All THREADS threads call it; `scratch` is
// shared memory of DEC_SCRATCH_INTS.  Ends with a block barrier.
template <int THREADS>
__device__ __forceinline__ DecWalk dec_walk_init(const int32_t* lengths, int nbh, int capacity, int mts, int extra, int cta,
                                                 int nctas, int* scratch) {
  int first, last, start;
  const DecLayout d = dec_layout<THREADS>(lengths, nbh, capacity, mts, extra, nctas, scratch, first, last, start);
  const int lo = min(d.total, cta * d.per);
  for (int i = first; i < last; ++i) {
    const int n = mts * ((cache_length(lengths, i, capacity) + DEC_TILE - 1) / DEC_TILE + 1 + d.extra);
    if (start <= lo && lo < start + n) {
      scratch[33] = i;
      scratch[34] = lo - start;
    }
    start += n;
  }
  __syncthreads();
  DecWalk walk;
  walk.lengths = lengths;
  walk.capacity = capacity;
  walk.mts = mts;
  walk.extra = d.extra;
  walk.left = min(d.per, d.total - lo);
  walk.bh = walk.left > 0 ? scratch[33] : 0;
  walk.unit = walk.left > 0 ? scratch[34] : 0;
  return walk;
}

// Bytes of the 16-byte chunk `chunk` (8 elements) of row r in a 128-byte-swizzled
// K-major tile whose 64-column groups are `group_bytes` apart.
__device__ __forceinline__ uint32_t sw128_offset(int r, int chunk, int group_bytes) {
  return static_cast<uint32_t>((chunk >> 3) * group_bytes + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
}

// Eight consecutive channels of a row of 16-bit elements, zero past `channels`,
// read one by one (rows that are not on 16 bytes).
__device__ __forceinline__ uint4 load_row_chunk(const uint16_t* row, int chunk, int channels) {
  const int c = chunk * 8;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = c + 2 * i < channels ? row[c + 2 * i] : 0u;
    const uint32_t hi = c + 2 * i + 1 < channels ? row[c + 2 * i + 1] : 0u;
    w[i] = lo | (hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Asynchronous 16-byte copy from global to shared memory; live == false fills
// zeros (src must still be a valid address).
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(live ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Bits of up to 32 mask bytes (1 where nonzero).  vec: 16-byte aligned, n a
// multiple of 16; otherwise all bytes are loaded before the first is used.
__device__ __forceinline__ uint32_t mask_word(const uint8_t* row, int n, bool vec) {
  uint32_t v = 0u;
  if (vec) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (16 * u >= n) continue;
      const uint4 x = reinterpret_cast<const uint4*>(row)[u];
      // Four mask bytes to four bits: 1 where nonzero, gathered by a multiply.
      v |= ((__vsetgtu4(x.x, 0u) * 0x01020408u) >> 24) << (16 * u);
      v |= ((__vsetgtu4(x.y, 0u) * 0x01020408u) >> 24) << (16 * u + 4);
      v |= ((__vsetgtu4(x.z, 0u) * 0x01020408u) >> 24) << (16 * u + 8);
      v |= ((__vsetgtu4(x.w, 0u) * 0x01020408u) >> 24) << (16 * u + 12);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < n) v |= (row[j] != 0 ? 1u : 0u) << j;
  }
  return v;
}

// The lowest n bits, 0 <= n <= 32.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

template <bool BF16>
__device__ __forceinline__ float elem_to_float(uint16_t x) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(x) << 16);
  else return __half2float(__ushort_as_half(x));
}

// Programmatic dependent launch: let the next kernel of the stream start (its
// prologue only), and wait until the previous ones are done and their writes
// are seen.  Every decode kernel is launched so and touches no memory before the
// wait, so whatever ran before it, decode kernel or not, it only overlaps that
// one's tail with its own start (barriers, TMEM, descriptors).  What they read is
// therefore not constant while they are resident, and a commit in place writes what
// it reads: none of it goes through the read-only path (__ldg), whose loads may
// also be moved ahead of the wait.
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace fe
