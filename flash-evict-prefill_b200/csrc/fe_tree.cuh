// Attention of drafted tokens over a cache (decode), for sm_100a.
//
// T drafted tokens per sequence (T = 1: an ordinary decode step) attend to the
// cached tokens of their row and to the drafts their tree mask names:
//   s = scale * q . [K_cache[0:n], K_new],  out = softmax(s) [V_cache; V_new],
//   lse = log sum exp s   (out 0 and lse -inf for a row that sees nothing).
//
// The G query heads of a KV head share its keys, so the G*T queries of one
// (b, hkv) are the rows of one matrix product: row g*T + t, in tiles of as many
// whole heads as fit the 128 TMEM lanes (one TMA box {64 channels, T, heads}).  What bounds it is reading K and V once (4*D bytes a
// cached token) until G*T reaches about 250 rows, then the tensor pipe; the
// padding of few rows to a 128-row MMA costs nothing that the memory time does
// not cover (1024 tensor cycles a tile against ~2800 cycles of HBM time an SM).
//
// Work: all rows' key tiles laid end to end, one equal run per SM
// (fe_decode.cuh), the last tile of a row being its drafts.  Each run leaves
// an unnormalised partial (O, m, l) per row it touched; fe_tree_join_kernel
// joins them in a fixed order (no atomics, bitwise reproducible).  Few short
// rows (a decode step over compacted caches) are latency instead: there a
// cluster of eight CTAs has a row and joins through distributed shared memory,
// in one launch (CLUSTER; 9.9 us for 4 rows of 2048, 11.3 the other way).
//
// Roles (384 threads): warps 0-3 and 4-7 are two softmax warpgroups, warp 8
// issues TMA, warp 9 tcgen05.mma.  Up to 128 rows (SPLIT) both warpgroups
// hold the same query tile and take alternate key tiles, each with its own S,
// O, m and l, so one's softmax hides the other's products; above 128 rows
// (DUAL) they hold two query tiles and both use every key tile.  Heads of more
// than 128 channels run one warpgroup (a 256-column O leaves no room for two).
#pragma once

#include <cooperative_groups.h>

#include "fe_decode.cuh"
#include "fe_forward.cuh"

namespace fe {

struct TreeParams {
  const uint16_t* q;
  int64_t q_sb, q_sh, q_st;  // strides in elements
  const uint16_t* k_new;
  int64_t kn_sb, kn_sh, kn_st;
  const uint16_t* v_new;
  int64_t vn_sb, vn_sh, vn_st;
  const uint8_t* tree;  // [T, T] per sequence, nonzero where draft t sees draft j; null: j <= t
  int64_t tree_sb;      // bytes between the sequences' masks (0: one mask for all)
  const int32_t* lengths;
  uint16_t* out;  // [B, Hq, T, D] contiguous
  float* lse;     // [B, Hq, T]
  float2* stats;  // workspace: [slots][R] {m, l}
  float4* acc;    // workspace: [slots][D4/4][R]: consecutive rows are consecutive in memory
  int B, Hq, Hkv, G, T, D, capacity;
  int M;             // G*T query rows of a KV head
  int tile_rows;     // of them in a 128-row tile: whole heads
  int MT, R, D4, nctas;
  float sc;  // scale * log2(e)
  uint64_t timeout_ns;
};

template <int DP, bool DUAL>
struct TreeCfg {
  static_assert(!DUAL || DP <= 128, "two query tiles need two O accumulators");
  static constexpr int NG = DP <= 128 ? 2 : 1;       // softmax warpgroups
  static constexpr bool SPLIT = NG == 2 && !DUAL;
  static constexpr int TILE = 128 * DP * 2;          // bytes of a 128-row tile
  static constexpr int NCH = DP / 64;
  static constexpr int QTILES = DUAL ? 2 : 1;
  static constexpr int STAGES = DP <= 64 ? 6 : (DP <= 128 ? (DUAL ? 2 : 3) : 1);
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = QTILES * TILE;
  static constexpr int OFF_V = OFF_K + STAGES * TILE;
  static constexpr int OFF_BAR = OFF_V + STAGES * TILE;
  // q_full[2], q_empty[2], k_full[S], v_full[S], k_empty[S], v_empty[S], s_full[2], p_full[2], o_full[2], drain
  static constexpr int NBAR = 4 + 4 * STAGES + 7;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int OFF_ML = OFF_MISC + 16 + 64 + DEC_SCRATCH_INTS * 4;  // float2[128]
  static constexpr int SMEM = OFF_ML + 128 * 8 + 1024;
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  static constexpr int THREADS = 384;
};

// The running maximum m is kept this far below the largest score (in powers of
// two), so P = 2^(s - m) is at most 2^(8 + 7) with the rescaling's slack.  In fp16
// that moves the weights that vanish, those under 2^-25, from 2^-25 of the row's
// largest to 2^-32: together below the output's own rounding for rows of up to 2^20
// tokens.  O, l and m carry the factor alike, so nothing else knows of it.  (bf16
// has FP32's range.)
template <bool BF16>
constexpr float TREE_HEADROOM = BF16 ? 0.0f : 7.0f;

// Lowest running max: finite, so that a row which has seen no key yet rescales
// by 2^-huge = 0 and never forms inf - inf.
constexpr float TREE_M0 = -3.0e38f;
// Key tiles that beginning and ending a row cost (batch of 16: 58.8 us with none,
// 56.1, 53.7, 53.1 and 53.7 with 1 to 4; 64 drafts over 32k 57.0, 54.9, 52.4, 52.4, 52.3).
constexpr int TREE_EXTRA = 3;
constexpr uint32_t TREE_QBUF = 8192;  // bytes between the halves of a query tile's 64-column group

// One key tile of a row's softmax (S in x).  With `masked`, only columns with
// their bit set count.  Lanes that hold no query (!live) have scores of whatever
// lay in the query tile: they follow the warp's rescaling and have no say in it.
template <bool BF16, int DV>
__device__ __forceinline__ void tree_softmax_tile(float (&x)[128], bool live, bool first, bool masked, const uint32_t (&bits)[4],
                                                  float sc, float sce, bool sc_pos, float& m_used, float& l,
                                                  uint32_t tS, uint32_t tO) {
  if (!sc_pos) {
#pragma unroll
    for (int c = 0; c < 128; ++c) x[c] *= sc;
  }
  if (masked) {
#pragma unroll
    for (int c = 0; c < 128; ++c) x[c] = ((bits[c >> 5] >> (c & 31)) & 1u) ? x[c] : -INFINITY;
  }
  const float m_new = fmaxf(m_used, row_max_scaled(x, sce) - TREE_HEADROOM<BF16>);
  if (first) {
    m_used = m_new;
  } else if (__any_sync(0xffffffffu, live && m_new > m_used + FWD_RESCALE_LOG2)) {
    // The product that last wrote O completed before this S did.
    const float f = ex2_approx(m_used - m_new);
    l *= f;
    m_used = m_new;
#pragma unroll 1
    for (int c0 = 0; c0 < DV; c0 += 32) {
      uint32_t o[32];
      tmem_ld32_sync(tO + c0, o);
#pragma unroll
      for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
      tmem_st32(tO + c0, o);
    }
    tmem_wait_st();
  }
  uint32_t pk[64];
  float amax;
  // P is rounded to the input type for the PV product (l sums it unrounded):
  // its error is that of one rounding per term, below the output's own, and in
  // fp16 at most 2^-32 of the row's largest weight where that is more.
  l += softmax_exp_pass<BF16, 0, false, 0>(x, sce, m_used, pk, amax);
  tmem_st32(tS, pk);
  tmem_st32(tS + 32, pk + 32);
  tmem_wait_st();
}

// Bits of the mask bytes [0, n), n <= 32 (1 where nonzero), in every lane of the
// warp.  A lane reads one byte.
__device__ __forceinline__ uint32_t tree_word(const uint8_t* row, int n) {
  const int lane = threadIdx.x & 31;
  const bool see = lane < n && row[lane] != 0;
  return __ballot_sync(0xffffffffu, see);
}

// bits: which of the 128 drafts draft t sees.  WARPS warps (`warp` of them this
// one), which meet at barrier `bar`, read the mask once, 64 drafts at a time,
// into `table` (two words a draft); each thread then takes its own row.  The
// rows of a tile's heads share drafts, so a thread reading its own row would
// read each byte once a head, on a line of its own (16 x 32 heads of 23 drafts
// after one token: 39.8 us so, 32.3 this way; 32 heads of 5 after 125 8.9, 7.4).
template <int WARPS>
__device__ __forceinline__ void tree_bits(const TreeParams& p, int b, int t, int warp, int bar, uint2* table,
                                          uint32_t (&bits)[4]) {
  if (p.tree == nullptr) {
#pragma unroll
    for (int w = 0; w < 4; ++w) bits[w] = low_bits(min(max(t + 1 - 32 * w, 0), 32));
    return;
  }
  const uint8_t* mask = p.tree + b * p.tree_sb;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int n = p.T - 64 * half;
    uint2 own = make_uint2(0u, 0u);
    if (n > 0) {
      named_bar_sync(bar, WARPS * 32);  // (everyone has taken what the table held)
#pragma unroll 4
      for (int row = warp; row < p.T; row += WARPS) {
        const uint8_t* at = mask + static_cast<int64_t>(row) * p.T + 64 * half;
        const uint32_t lo = tree_word(at, min(n, 32)), hi = tree_word(at + 32, min(max(n - 32, 0), 32));
        if ((threadIdx.x & 31) == 0) table[row] = make_uint2(lo, hi);
      }
      named_bar_sync(bar, WARPS * 32);
      own = table[t];
    }
    bits[2 * half] = own.x;
    bits[2 * half + 1] = own.y;
  }
}

// Adds the weighted value rows of the drafts in `bits`, whose V rows are not
// finite and were left out of the product, to one row's partial O in memory:
// only rows that see such a draft come here (see the draft tile).
template <bool BF16>
__device__ __noinline__ void tree_add_special(const TreeParams& p, int b, int h, int g, int t, uint32_t bits, int j0,
                                              float m, float4* o) {
  const uint16_t* q = p.q + b * p.q_sb + (static_cast<int64_t>(h) * p.G + g) * p.q_sh + t * p.q_st;
  for (; bits != 0u; bits &= bits - 1u) {
    const int j = j0 + __ffs(bits) - 1;
    const uint16_t* k = p.k_new + b * p.kn_sb + h * p.kn_sh + j * p.kn_st;
    const uint16_t* v = p.v_new + b * p.vn_sb + h * p.vn_sh + j * p.vn_st;
    float s = 0.f;
    for (int d = 0; d < p.D; ++d) s = fmaf(elem_to_float<BF16>(q[d]), elem_to_float<BF16>(k[d]), s);
    const float w = ex2_approx(s * p.sc - m);
    for (int c = 0; c < p.D; ++c) reinterpret_cast<float*>(o + (c >> 2) * p.R)[c & 3] += w * elem_to_float<BF16>(v[c]);
  }
}

// Nonzero if one of two packed 16-bit values has all exponent bits set.
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
  constexpr uint32_t E = BF16 ? 0x7f807f80u : 0x7c007c00u;
  return __vcmpeq2(w & E, E);
}

constexpr int TREE_CLUSTER = 8;

// Running combination of partials of one row: four channels per quad.
template <int Q>
struct TreeMerge {
  float m, l;
  float4 a[Q];
  __device__ __forceinline__ void init() {
    m = TREE_M0;
    l = 0.f;
#pragma unroll
    for (int j = 0; j < Q; ++j) a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void add(float2 st, const float4 (&v)[Q]) {
    if (st.y == 0.f) return;  // this part saw no key of the row: its O may not have been written
    const float mn = fmaxf(m, st.x);
    const float f = exp2f(m - mn), g = exp2f(st.x - mn);
    m = mn;
    l = l * f + st.y * g;
#pragma unroll
    for (int j = 0; j < Q; ++j) {
      a[j].x = a[j].x * f + v[j].x * g;
      a[j].y = a[j].y * f + v[j].y * g;
      a[j].z = a[j].z * f + v[j].z * g;
      a[j].w = a[j].w * f + v[j].w * g;
    }
  }
  // Writes the row's channels [quad0*4, ...) and, with the first of them, its lse.
  template <bool BF16>
  __device__ __forceinline__ void store(const TreeParams& p, int64_t orow, int quad0) const {
    const bool none = l == 0.f;
    const float inv = none ? 0.f : 1.0f / l;
    uint16_t* out = p.out + orow * p.D;
#pragma unroll
    for (int j = 0; j < Q; ++j) {
      const int c = (quad0 + j) * 4;
      if (c >= p.D) continue;
      const uint32_t lo = pack2<BF16>(a[j].x * inv, a[j].y * inv), hi = pack2<BF16>(a[j].z * inv, a[j].w * inv);
      if ((p.D & 3) == 0) {
        *reinterpret_cast<uint2*>(out + c) = make_uint2(lo, hi);
      } else {
        const uint16_t w[4] = {static_cast<uint16_t>(lo), static_cast<uint16_t>(lo >> 16), static_cast<uint16_t>(hi),
                               static_cast<uint16_t>(hi >> 16)};
        for (int i = 0; i < 4 && c + i < p.D; ++i) out[c + i] = w[i];
      }
    }
    if (quad0 == 0) p.lse[orow] = none ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
  }
};

// All threads of the cluster, each warp converged; the roles meet here from
// different places.
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <bool BF16, int DP, bool DUAL, bool CLUSTER>
__global__ void __launch_bounds__(384, 1)
    fe_tree_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                   const __grid_constant__ CUtensorMap tv,
                   const __grid_constant__ CUtensorMap tkn, const __grid_constant__ CUtensorMap tvn,
                   const __grid_constant__ TreeParams p) {
  using C = TreeCfg<DP, DUAL>;
  constexpr int NG = C::NG;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_empty = q_full + 2;
  uint64_t* k_full = q_empty + 2;
  uint64_t* v_full = k_full + C::STAGES;
  uint64_t* k_empty = v_full + C::STAGES;
  uint64_t* v_empty = k_empty + C::STAGES;
  uint64_t* s_full = v_empty + C::STAGES;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* drain = o_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  // Drafts whose V row is not finite, 128 bits: [group that took the draft tile][segment parity].
  uint32_t* special = tmem_holder + 4;
  int* scratch = reinterpret_cast<int*>(special + 16);

  float2* s_ml = reinterpret_cast<float2*>(smem + C::OFF_ML);

  const int warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 256) {
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
    tma_prefetch_desc(&tkn);
    tma_prefetch_desc(&tvn);
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  if (warp == 9) {
    __syncwarp();
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  pdl_wait();  // nothing above reads or writes memory
  DecWalk walk;
  if constexpr (CLUSTER) {
    // A CTA of the cluster has an eighth of one item's tiles.
    const int item = blockIdx.x / TREE_CLUSTER, rank = blockIdx.x % TREE_CLUSTER;
    walk.lengths = p.lengths;
    walk.capacity = p.capacity;
    walk.mts = p.MT;
    walk.extra = 0;
    walk.bh = item / p.MT;
    const int tiles = (cache_length(p.lengths, walk.bh, p.capacity) + DEC_TILE - 1) / DEC_TILE + 1;
    const int share = (tiles + TREE_CLUSTER - 1) / TREE_CLUSTER, j0 = min(rank * share, tiles);
    walk.left = min(share, tiles - j0);
    walk.unit = (item - walk.bh * p.MT) * tiles + j0;
    if (threadIdx.x == 0) scratch[0] = (tiles + share - 1) / share;  // CTAs that have tiles
    __syncthreads();
  } else {
    // Ends with a block barrier, which also publishes the barriers and TMEM.
    walk = dec_walk_init<C::THREADS>(p.lengths, p.B * p.Hkv, p.capacity, p.MT, TREE_EXTRA, blockIdx.x, p.nctas, scratch);
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const uint64_t TO = p.timeout_ns;
  // Query tiles of at most 64 rows are double-buffered in the two halves of
  // the tile, so a run's next row starts while the last one is written out.  The
  // MMA reads 128 rows all the same: the others' scores stay on their own TMEM
  // lanes, which nobody reads.
  const uint32_t qbufs = !DUAL && p.tile_rows <= 64 ? 2 : 1;
  DecSegment sg;

  if (warp >= 8) {
    setmaxnreg_dec<FWD_REGS_LOW>();
    if (warp == 8) {
      // ---------------------------------------------------------- producer --
      if (lane == 0) {
        uint32_t loads[C::STAGES];
        for (int s = 0; s < C::STAGES; ++s) loads[s] = 0;
        bool ok = true;
        uint32_t it = 0, nseg = 0;
        const int heads = p.tile_rows / p.T;  // per query tile
        while (ok && walk.next(sg)) {
          const int b = sg.bh / p.Hkv, h = sg.bh - b * p.Hkv;
          // The segment's queries: whole heads, their rows one after another.
          // (Rows past the last head of the KV head are read and not used.)
          const uint32_t qb = nseg % qbufs, quse = nseg / qbufs;
          if (quse > 0) ok = mbar_wait(&q_empty[qb], (quse - 1) & 1, TO, abort_flag);
          if (!ok) break;
          mbar_expect_tx(&q_full[qb], C::QTILES * p.tile_rows * DP * 2);
          for (int t = 0; t < C::QTILES; ++t)
            for (int c = 0; c < C::NCH; ++c)
              tma_load_4d(smem + C::OFF_Q + t * C::TILE + c * 16384 + qb * TREE_QBUF, &tq, &q_full[qb], c * 64, 0,
                          h * p.G + (sg.mt * C::QTILES + t) * heads, b);
          ++nseg;
          for (int j = sg.j0; j < sg.j1; ++j, ++it) {
            const int s = it % C::STAGES;
            const uint32_t use = it / C::STAGES;
            const bool drafts = j == sg.tiles - 1;
            const CUtensorMap* mk = drafts ? &tkn : &tk;
            const CUtensorMap* mv = drafts ? &tvn : &tv;
            const int row = drafts ? 0 : j * DEC_TILE;
            if (use > 0) ok = mbar_wait(&k_empty[s], (use - 1) & 1, TO, abort_flag);
            if (!ok) break;
            mbar_expect_tx(&k_full[s], C::TILE);
            for (int c = 0; c < C::NCH; ++c)
              tma_load_4d(smem + C::OFF_K + s * C::TILE + c * 16384, mk, &k_full[s], c * 64, row, h, b);
            if (use > 0) ok = mbar_wait(&v_empty[s], (use - 1) & 1, TO, abort_flag);
            if (!ok) {
              loads[s] = use * 2 + 1;  // K of this use in flight, V not issued
              break;
            }
            mbar_expect_tx(&v_full[s], C::TILE);
            for (int c = 0; c < C::NCH; ++c)
              tma_load_4d(smem + C::OFF_V + s * C::TILE + c * 16384, mv, &v_full[s], c * 64, row, h, b);
            loads[s] = use * 2 + 2;
          }
        }
        // Never leave the CTA with a TMA write in flight.
        for (uint32_t i = nseg > qbufs ? nseg - qbufs : 0; i < nseg; ++i)
          mbar_wait_inflight(&q_full[i % qbufs], (i / qbufs) & 1, TO);
        for (int s = 0; s < C::STAGES; ++s) {
          if (loads[s] == 0) continue;
          const uint32_t use = (loads[s] - 1) / 2;
          mbar_wait_inflight(&k_full[s], use & 1, TO);
          if (loads[s] % 2 == 0) mbar_wait_inflight(&v_full[s], use & 1, TO);
        }
      }
    } else if (warp == 9) {
      // -------------------------------------------------------- MMA issuer --
      // Step i of a segment is one (query tile, key tile): group i % NG; key
      // tile i in SPLIT, i / 2 in DUAL.  Order: S(0), S(1), then PV(i),
      // S(i + NG) -- so when a group sees S complete, its previous PV is too.
      if (lane == 0) {
        constexpr uint32_t ID_S = idesc_f16(128, 128, BF16, false);
        constexpr uint32_t ID_PV = idesc_f16(128, DP, BF16, true);
        const uint64_t dq = smem_desc_sw128(smem_u32(smem + C::OFF_Q), 16, 1024);
        const uint64_t dk = smem_desc_sw128(smem_u32(smem + C::OFF_K), 16, 1024);
        const uint64_t dv = smem_desc_sw128(smem_u32(smem + C::OFF_V), 16384, 1024);
        const uint32_t dq_lo = static_cast<uint32_t>(dq), dq_hi = static_cast<uint32_t>(dq >> 32);
        const uint32_t dk_lo = static_cast<uint32_t>(dk), dk_hi = static_cast<uint32_t>(dk >> 32);
        const uint32_t dv_lo = static_cast<uint32_t>(dv), dv_hi = static_cast<uint32_t>(dv >> 32);
        constexpr uint32_t TILE16 = C::TILE >> 4;
        uint32_t it0 = 0;           // key tiles of the segments before
        uint32_t nseg = 0;
        uint32_t np[2] = {0, 0};    // P tiles consumed per group
        bool ok = true;
        while (ok && walk.next(sg)) {
          const int ntile = sg.j1 - sg.j0;
          const int steps = DUAL ? 2 * ntile : ntile;
          const uint32_t qb = nseg % qbufs;
          auto tile_of = [&](int i) { return it0 + static_cast<uint32_t>(DUAL ? i >> 1 : i); };
          auto issue_s = [&](int i) -> bool {
            const uint32_t tile = tile_of(i);
            const int s = tile % C::STAGES, t = i % NG;
            if (!DUAL || (i & 1) == 0) {
              if (!mbar_wait(&k_full[s], (tile / C::STAGES) & 1, TO, abort_flag)) return false;
              tc_fence_after();
            }
            const uint32_t a = dq_lo + (DUAL ? t * TILE16 : qb * (TREE_QBUF >> 4));
            const uint32_t bb = dk_lo + s * TILE16;
#pragma unroll 8
            for (int kk = 0; kk < DP / 16; ++kk) {
              const uint32_t off = static_cast<uint32_t>(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4);
              umma_ss_lohi(tmem + t * 128, a + off, dq_hi, bb + off, dk_hi, ID_S, kk > 0);
            }
            umma_commit(&s_full[t]);
            if (!DUAL || (i & 1) == 1) umma_commit(&k_empty[s]);
            if (i == steps - 1) umma_commit(&q_empty[qb]);
            return true;
          };
          ok = mbar_wait(&q_full[qb], (nseg / qbufs) & 1, TO, abort_flag);
          if (!ok) break;
          tc_fence_after();
          for (int i = 0; i < NG && i < steps && ok; ++i) ok = issue_s(i);
          for (int i = 0; i < steps && ok; ++i) {
            const uint32_t tile = tile_of(i);
            const int s = tile % C::STAGES, t = i % NG;
            if (!DUAL || (i & 1) == 0) ok = mbar_wait(&v_full[s], (tile / C::STAGES) & 1, TO, abort_flag);
            if (ok) ok = mbar_wait(&p_full[t], np[t] & 1, TO, abort_flag);
            if (!ok) break;
            ++np[t];
            tc_fence_after();
            const uint32_t bb = dv_lo + s * TILE16;
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              umma_ts_lohi(tmem + 128 * NG + t * DP, tmem + t * 128 + kk * 8, bb + static_cast<uint32_t>(kk * 128),
                           dv_hi, ID_PV, (i >= NG || kk > 0) ? 1u : 0u);
            if (!DUAL || (i & 1) == 1) umma_commit(&v_empty[s]);
            if (i + NG < steps) ok = issue_s(i + NG);
            else umma_commit(&o_full[t]);
          }
          if (ok && steps < NG) umma_commit(&o_full[1]);  // one commit a segment for a group without a step, too
          it0 += ntile;
          ++nseg;
        }
        umma_commit(drain);
        mbar_wait_inflight(drain, 0, TO);
      }
    }
    if constexpr (CLUSTER) {
      cluster_barrier();
      cluster_barrier();
    }
  } else {
    setmaxnreg_inc<FWD_REGS_HIGH>();
    // ------------------------------------------------------------- softmax --
    const int t = warp >> 2;
    if (t < NG) {
      const int r = ((warp & 3) << 5) + static_cast<int>(lane);  // TMEM lane
      const uint32_t lane_off = static_cast<uint32_t>((warp & 3) << 5) << 16;
      const uint32_t tS = tmem + lane_off + t * 128;
      const uint32_t tO = tmem + lane_off + 128 * NG + t * DP;
      const float sc = p.sc;
      const bool sc_pos = sc > 0.f;
      const float sce = sc_pos ? sc : 1.0f;
      // CLUSTER: the partial stays in shared memory, O in the place of the tiles
      // (every load has landed and every product has read them by then; after an
      // abort it may be overwritten, but not the NaN statistics in s_ml).
      float4* s_part = reinterpret_cast<float4*>(smem);
      bool ok = true;
      uint32_t it0 = 0, nseg = 0, ns = 0;  // key tiles before, segments, S tiles of this group
      for (; walk.next(sg); ++nseg) {
        const int b = sg.bh / p.Hkv, h = sg.bh - b * p.Hkv;
        const int ntile = sg.j1 - sg.j0;
        const int pr = (DUAL ? t * p.tile_rows : 0) + r;  // row of the item
        const int row = sg.mt * C::QTILES * p.tile_rows + pr;  // of the KV head's G*T queries
        const bool live = r < p.tile_rows && row < p.M;
        const bool warp_live = __any_sync(0xffffffffu, live);
        const int g = live ? row / p.T : 0, tt = live ? row - g * p.T : 0;
        // Who takes the draft tile notes which drafts its rows see, and starts a
        // clean list of drafts that need special care.
        const bool has_drafts = sg.j1 == sg.tiles;
        const int owner = DUAL ? 0 : (ntile - 1) % NG;  // group that takes the last tile (DUAL: that clears its V rows)
        const bool mine = has_drafts && (DUAL || owner == t);
        uint32_t* spec = special + owner * 8 + (nseg & 1) * 4;
        uint32_t bits[4] = {0u, 0u, 0u, 0u};
        if (mine) {
          // s_ml is free until the segment's end: SPLIT's other warpgroup writes it
          // after its O, whose last product is issued after this group's first P.
          tree_bits<DUAL ? 8 : 4>(p, b, tt, DUAL ? warp : warp & 3, DUAL ? 3 : 1 + t, reinterpret_cast<uint2*>(s_ml), bits);
          if (!live) bits[0] = bits[1] = bits[2] = bits[3] = 0u;
          // Nobody reads this list any more: two segments back, both groups of two
          // query tiles did (SPLIT's groups meet at every segment's end).
          if constexpr (DUAL) named_bar_sync(3, 256);
          if (t == owner) {
            if constexpr (!DUAL) named_bar_sync(1 + t, 128);
            if (r < 4) spec[r] = 0u;
            named_bar_sync(1 + t, 128);
          }
        }
        float m_used = TREE_M0, l = 0.f;
        bool first = true;
        for (int i = DUAL ? 0 : t; i < ntile && ok; i += DUAL ? 1 : NG) {
          const int j = sg.j0 + i;
          const uint32_t tile = it0 + i;
          const int s = tile % C::STAGES;
          ok = warp_all(mbar_wait(&s_full[t], ns & 1, TO, abort_flag));
          if (!ok) break;
          ++ns;
          tc_fence_after();
          const bool drafts = j == sg.tiles - 1;
          const int lim = drafts ? p.T - 1 : sg.len - 1 - j * DEC_TILE;
          if ((drafts || lim < 127) && (!DUAL || t == 0)) {
            // A masked column's P is 0, but 0 * V must be 0 too: slots past the
            // length hold anything, and a draft's V row may not be finite.
            // Clear those rows (thread = V row) before the product reads them.
            ok = warp_all(mbar_wait(&v_full[s], (tile / C::STAGES) & 1, TO, abort_flag));
            if (!ok) break;
            // (Rows past the drafts were filled with zeros by the load.)
            uint8_t* vt = smem + C::OFF_V + s * C::TILE + r * 128;
            bool clear = r > lim && !drafts;
            if (drafts && r <= lim) {
              uint32_t bad = 0u;
#pragma unroll
              for (int c = 0; c < C::NCH; ++c)
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                  const uint4 w = *reinterpret_cast<const uint4*>(vt + c * 16384 + (u << 4));
                  bad |= not_finite2<BF16>(w.x) | not_finite2<BF16>(w.y) | not_finite2<BF16>(w.z) | not_finite2<BF16>(w.w);
                }
              clear = bad != 0u;
              if (clear) atomicOr(&spec[r >> 5], 1u << (r & 31));
            }
            if (__any_sync(0xffffffffu, clear)) {
              for (int c = 0; c < C::NCH && clear; ++c)
#pragma unroll
                for (int u = 0; u < 8; ++u)
                  *reinterpret_cast<uint4*>(vt + c * 16384 + ((u ^ (r & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
              fence_proxy_async_smem();
            }
          }
          if (warp_live) {
            float x[128];
            {
              uint32_t* xr = reinterpret_cast<uint32_t*>(x);
              tmem_ld64_sync(tS, xr);
              tmem_ld64_sync(tS + 64, xr + 64);
            }
            uint32_t sees[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              sees[w] = drafts ? bits[w] : low_bits(min(max(lim + 1 - 32 * w, 0), 32));
            }
            const bool masked = drafts || lim < 127;
            if (DUAL && !masked)  // the long runs' loop, free of masking code
              tree_softmax_tile<BF16, DP>(x, live, first, false, sees, sc, sce, sc_pos, m_used, l, tS, tO);
            else
              tree_softmax_tile<BF16, DP>(x, live, first, masked, sees, sc, sce, sc_pos, m_used, l, tS, tO);
          }
          first = false;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[t]);
        }
        if (ok) ok = warp_all(mbar_wait(&o_full[t], nseg & 1, TO, abort_flag));
        tc_fence_after();
        // ---- result of this run for the row: a partial, or the row itself
        // when the run has all of its tiles
        const bool whole = !CLUSTER && sg.j0 == 0 && sg.j1 == sg.tiles;
        const float nan = __int_as_float(0x7fffffff);
        float f0 = 1.f, f1 = 0.f;  // weights of O of this group's lanes, and (SPLIT) of the other warpgroup's
        if (!ok) m_used = l = nan;  // aborted (watchdog): everything below becomes NaN
        if constexpr (C::SPLIT) {
          // Both warpgroups hold the row (lane r of two O tiles); each writes
          // half of the channels of their sum.
          const float2 own = make_float2(m_used, l);
          if (t == 1) s_ml[r] = own;
          named_bar_sync(3, 256);
          float2 a = own, c = own;
          if (t == 0) {
            c = s_ml[r];
            s_ml[r] = own;
          }
          named_bar_sync(3, 256);
          if (t == 1) a = s_ml[r];
          m_used = fmaxf(a.x, c.x);
          f0 = ex2_approx(a.x - m_used);
          f1 = ex2_approx(c.x - m_used);
          l = a.y * f0 + c.y * f1;
        }
        const bool two = C::SPLIT && ntile > 1;
        const int64_t slot = static_cast<int64_t>(sg.bh) * p.MT + sg.mt + blockIdx.x;
        const int64_t orow = static_cast<int64_t>(sg.bh) * p.M + row;
        float4* dst = CLUSTER ? s_part + pr : p.acc + slot * p.R * (p.D4 / 4) + pr;
        uint16_t* out = p.out + orow * p.D;
        // Special rows are added in memory, so such a run's sum goes through it.
        const bool special_rows = has_drafts && (spec[0] | spec[1] | spec[2] | spec[3]) != 0u;
        const bool direct = whole && !special_rows;
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        if (live && (!C::SPLIT || t == 0)) {
          if (whole) p.lse[orow] = l == 0.f ? -INFINITY : (m_used + log2f(l)) * 0.69314718055994531f;
          else if (!CLUSTER) p.stats[slot * p.R + pr] = make_float2(m_used, l);
        }
        if (warp_live) {
          constexpr int CB = C::SPLIT ? DP / 2 : DP;
#pragma unroll 1
          for (int c0 = C::SPLIT ? t * CB : 0; c0 < (C::SPLIT ? (t + 1) * CB : DP); c0 += 32) {
            uint32_t o[32];
            tmem_ld32_sync((C::SPLIT ? tO - t * DP : tO) + c0, o);
            if (two) {
              uint32_t o1[32];
              tmem_ld32_sync(tO - t * DP + DP + c0, o1);
#pragma unroll
              for (int c = 0; c < 32; ++c)
                o[c] = __float_as_uint(__uint_as_float(o[c]) * f0 + __uint_as_float(o1[c]) * f1);
            }
            if (live && direct) {
#pragma unroll
              for (int c = 0; c < 32; c += 8) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  w[e] = pack2<BF16>(__uint_as_float(o[c + 2 * e]) * inv, __uint_as_float(o[c + 2 * e + 1]) * inv);
                if ((p.D & 7) == 0) {
                  if (c0 + c < p.D) *reinterpret_cast<uint4*>(out + c0 + c) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
#pragma unroll
                  for (int e = 0; e < 8; ++e)
                    if (c0 + c + e < p.D) out[c0 + c + e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
                }
              }
            } else if (live) {
#pragma unroll
              for (int q4 = 0; q4 < 8; ++q4)
                if (c0 + q4 * 4 < p.D4)
                  *reinterpret_cast<uint4*>(dst + (c0 / 4 + q4) * p.R) =
                      make_uint4(o[4 * q4], o[4 * q4 + 1], o[4 * q4 + 2], o[4 * q4 + 3]);
            }
          }
        }
        if (special_rows) {
          if constexpr (C::SPLIT) named_bar_sync(3, 256);
          if (mine && live) {
#pragma unroll
            for (int w = 0; w < 4; ++w) tree_add_special<BF16>(p, b, h, g, tt, bits[w] & spec[w], 32 * w, m_used, dst);
            if (whole)
              for (int c = 0; c < p.D; ++c)
                out[c] = static_cast<uint16_t>(pack2<BF16>(reinterpret_cast<float*>(dst + (c >> 2) * p.R)[c & 3] * inv, 0.f));
          }
        }
        tc_fence_before();
        if constexpr (C::SPLIT) named_bar_sync(3, 256);  // both are done with both O tiles and with s_ml
        if (CLUSTER && t == 0) s_ml[r] = make_float2(m_used, l);
        it0 += ntile;
      }
    }
    if constexpr (CLUSTER) {
      cluster_barrier();
      // Every CTA joins an eighth of the item's rows and channels, both
      // warpgroups, from the CTAs that had tiles.
      cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
      const float4* s_part = reinterpret_cast<const float4*>(smem);
      const int item = blockIdx.x / TREE_CLUSTER, rank = blockIdx.x % TREE_CLUSTER;
      const int bh = item / p.MT, mt = item - bh * p.MT;
      const int used = scratch[0];
      const int rows = min(p.M - mt * p.tile_rows, p.tile_rows), pairs = rows * (p.D4 / 4);
      const int share = (pairs + TREE_CLUSTER - 1) / TREE_CLUSTER, end = min(pairs, (rank + 1) * share);
      for (int i = rank * share + static_cast<int>(threadIdx.x); i < end; i += 256) {
        const int quad = i / rows, rr = i - quad * rows;
        float2 st[TREE_CLUSTER];
        float4 v[TREE_CLUSTER][1];
#pragma unroll
        for (int c = 0; c < TREE_CLUSTER; ++c)
          if (c < used) {
            st[c] = *cluster.map_shared_rank(s_ml + rr, c);
            v[c][0] = *cluster.map_shared_rank(s_part + quad * p.R + rr, c);
          }
        TreeMerge<1> sum;
        sum.init();
#pragma unroll
        for (int c = 0; c < TREE_CLUSTER; ++c)
          if (c < used) sum.add(st[c], v[c]);
        sum.template store<BF16>(p, static_cast<int64_t>(bh) * p.M + mt * p.tile_rows + rr, quad);
      }
      cluster_barrier();  // nobody leaves while a neighbour reads its partial
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

constexpr int TREE_JOIN_THREADS = 256;
constexpr int TREE_JOIN_WARPS = TREE_JOIN_THREADS / 32;
constexpr int TREE_JOIN_QUADS = 4;  // channel quads per thread

// Joins the runs' partials of a row.  A thread owns 16 channels of one row
// (consecutive threads: consecutive rows, as the partials lie) and merges
// every splits-th partial with a running maximum; the `splits` warps that share
// a set of rows are merged through shared memory in a fixed order.
template <bool BF16>
__global__ void __launch_bounds__(TREE_JOIN_THREADS)
    fe_tree_join_kernel(const __grid_constant__ TreeParams p, int rows_per_item, int splits) {
  constexpr int Q = TREE_JOIN_QUADS;
  __shared__ float4 s_acc[TREE_JOIN_WARPS][Q][32];
  __shared__ float2 s_ml[TREE_JOIN_WARPS][32];
  __shared__ int scratch[TREE_JOIN_WARPS], s_start;
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int split = warp % splits;
  const int quads = p.D4 / 4, groups = (quads + Q - 1) / Q;
  const int item = blockIdx.x;
  const int bh = item / p.MT, mt = item - bh * p.MT;
  const int rows = min(p.M - mt * rows_per_item, rows_per_item);
  const int pair = (blockIdx.y * (TREE_JOIN_WARPS / splits) + warp / splits) * 32 + lane;
  const bool live = pair < rows * groups;
  const int quad0 = live ? pair / rows * Q : 0, r = live ? pair % rows : 0;
  // Which runs had the row.  (The kernel before the attention may have written
  // the lengths and still be running until here: the attention lets this one
  // start ahead of its own wait.  Of 64 drafts over 32k, 52.4 us, it costs about 1.)
  pdl_wait();
  int first, last, start;
  const DecLayout d = dec_layout<TREE_JOIN_THREADS>(p.lengths, p.B * p.Hkv, p.capacity, p.MT, TREE_EXTRA, p.nctas, scratch,
                                                    first, last, start);
  for (int i = first; i < last && i <= bh; ++i) {
    if (i == bh) s_start = start;
    start += p.MT * ((cache_length(p.lengths, i, p.capacity) + DEC_TILE - 1) / DEC_TILE + 1 + d.extra);
  }
  __syncthreads();
  const int tiles = (cache_length(p.lengths, bh, p.capacity) + DEC_TILE - 1) / DEC_TILE + 1;
  const int u0 = s_start + mt * (tiles + d.extra);
  const int c0 = u0 / d.per, n = (u0 + tiles - 1) / d.per - c0 + 1;
  if (n == 1) return;  // one run had the whole row and wrote it
  const int64_t slot0 = static_cast<int64_t>(item) + c0;
  const float2* st_row = p.stats + slot0 * p.R + r;
  const float4* acc_row = p.acc + slot0 * p.R * quads + static_cast<int64_t>(quad0) * p.R + r;
  const int64_t acc_step = static_cast<int64_t>(p.R) * quads;
  TreeMerge<Q> sum;
  sum.init();
  if (live) {
    constexpr int U = 3;
    for (int i0 = split; i0 < n; i0 += splits * U) {
      float2 st[U];
      float4 v[U][Q];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * splits;
        st[u] = make_float2(0.f, 0.f);
        if (i < n) {
          st[u] = __ldcs(st_row + static_cast<int64_t>(i) * p.R);
#pragma unroll
          for (int j = 0; j < Q; ++j)
            if (quad0 + j < quads) v[u][j] = __ldcs(acc_row + i * acc_step + j * p.R);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) sum.add(st[u], v[u]);
    }
  }
  if (splits > 1) {
    s_ml[warp][lane] = make_float2(sum.m, sum.l);
#pragma unroll
    for (int j = 0; j < Q; ++j) s_acc[warp][j][lane] = sum.a[j];
    __syncthreads();
    if (split != 0) return;
    for (int w = 1; w < splits; ++w) {
      float4 v[Q];
#pragma unroll
      for (int j = 0; j < Q; ++j) v[j] = s_acc[warp + w][j][lane];
      sum.add(s_ml[warp + w][lane], v);
    }
  }
  if (live) sum.template store<BF16>(p, static_cast<int64_t>(bh) * p.M + mt * rows_per_item + r, quad0);
}

}  // namespace fe
