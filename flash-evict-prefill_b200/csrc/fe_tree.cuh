// Attention of drafted tokens over a cache (decode), for sm_100a.
//
// T drafted tokens per sequence (T = 1: an ordinary decode step) attend to the
// cached tokens of their row and to the drafts their tree mask names:
//   s = scale * q . [K_cache[0:n], K_new],  out = softmax(s) [V_cache; V_new],
//   lse = log sum exp s   (out 0 and lse -inf for a row that sees nothing).
//
// The G query heads of a KV head share its keys, so the G*T queries of one
// (b, hkv) are the rows of one matrix product: row r = g*T + t, tiles of 128
// rows on the TMEM lanes.  What bounds it is reading K and V once (4*D bytes a
// cached token) until G*T reaches about 250 rows, then the tensor pipe; the
// padding of few rows to a 128-row MMA costs nothing that the memory time does
// not cover (1024 tensor cycles a tile against ~2800 cycles of HBM time an SM).
//
// Work: all rows' key tiles laid end to end, one equal run per SM
// (fe_decode.cuh), the last tile of a row being its drafts.  Each run leaves
// an unnormalised partial (O, m, l) per row it touched; fe_tree_join_kernel
// joins them in a fixed order (no atomics, bitwise reproducible).
//
// Roles (384 threads): warps 0-3 and 4-7 are two softmax warpgroups, warp 8
// issues TMA, warp 9 tcgen05.mma.  Up to 128 rows (SPLIT) both warpgroups
// hold the same query tile and take alternate key tiles, each with its own S,
// O, m and l, so one's softmax hides the other's products; above 128 rows
// (DUAL) they hold two query tiles and both use every key tile.  Heads of more
// than 128 channels run one warpgroup (a 256-column O leaves no room for two).
#pragma once

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
  int32_t* base;  // workspace: first unit of every row, total
  float2* stats;  // workspace: [slots][groups][R] {m, l}
  float* acc;     // workspace: [slots][groups][R][D4]
  int B, Hq, Hkv, G, T, D, capacity;
  int M, MT, R, D4, nctas;
  float sc;  // scale * log2(e)
  int q_vec;
  uint64_t timeout_ns;
};

template <int DP, bool DUAL>
struct TreeCfg {
  static_assert(!DUAL || DP <= 128, "two query tiles need two O accumulators");
  static constexpr int NG = DP <= 128 ? 2 : 1;       // softmax warpgroups
  static constexpr int ROWS = DUAL ? 256 : 128;      // query rows per work item
  static constexpr int PARTS = (NG == 2 && !DUAL) ? 2 : 1;  // partials a run leaves per row
  static constexpr int TILE = 128 * DP * 2;          // bytes of a 128-row tile
  static constexpr int NCH = DP / 64;
  static constexpr int QTILES = DUAL ? 2 : 1;
  static constexpr int STAGES = DP <= 64 ? 6 : (DP <= 128 ? (DUAL ? 2 : 3) : 1);
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = QTILES * TILE;
  static constexpr int OFF_V = OFF_K + STAGES * TILE;
  static constexpr int OFF_BAR = OFF_V + STAGES * TILE;
  // q_full, k_full[S], v_full[S], k_empty[S], v_empty[S], s_full[2], p_full[2], o_full[2], drain
  static constexpr int NBAR = 1 + 4 * STAGES + 7;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM = OFF_MISC + 16 + 32 + DEC_SCRATCH_INTS * 4 + 1024;
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  static constexpr int THREADS = 384;
};

// Lowest running max: finite, so that a row which has seen no key yet rescales
// by 2^-huge = 0 and never forms inf - inf.
constexpr float TREE_M0 = -3.0e38f;

// One key tile of a row's softmax (S in x).  KIND 0: every column counts;
// 1: columns past lim do not; 2: only columns with their bit set do.
template <bool BF16, int DV, int KIND>
__device__ __forceinline__ void tree_softmax_tile(float (&x)[128], bool first, int lim, const uint32_t (&bits)[4],
                                                  float sc, float sce, bool sc_pos, float& m_used, float& l,
                                                  uint32_t tS, uint32_t tO) {
  if (!sc_pos) {
#pragma unroll
    for (int c = 0; c < 128; ++c) x[c] *= sc;
  }
  if constexpr (KIND == 1) {
#pragma unroll
    for (int c = 0; c < 128; ++c) x[c] = (c <= lim) ? x[c] : -INFINITY;
  }
  if constexpr (KIND == 2) {
#pragma unroll
    for (int c = 0; c < 128; ++c) x[c] = ((bits[c >> 5] >> (c & 31)) & 1u) ? x[c] : -INFINITY;
  }
  const float m_new = fmaxf(m_used, row_max_scaled(x, sce));
  if (first) {
    m_used = m_new;
  } else if (__any_sync(0xffffffffu, m_new > m_used + FWD_RESCALE_LOG2)) {
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
  // its error is that of one rounding per term, below the output's own.
  l += softmax_exp_pass<BF16, 0, false, 0>(x, sce, m_used, pk, amax);
  tmem_st32(tS, pk);
  tmem_st32(tS + 32, pk + 32);
  tmem_wait_st();
}

// Bit j of the 128: draft t sees draft j.
__device__ __forceinline__ void tree_bits(const TreeParams& p, int b, int t, uint32_t (&bits)[4]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) bits[w] = 0u;
  if (p.tree == nullptr) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int n = min(max(t + 1 - 32 * w, 0), 32);
      bits[w] = n == 32 ? 0xffffffffu : ((1u << n) - 1u);
    }
    return;
  }
  const uint8_t* row = p.tree + b * p.tree_sb + static_cast<int64_t>(t) * p.T;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int n = min(max(p.T - 32 * w, 0), 32);
    uint32_t v = 0u;
#pragma unroll 8
    for (int j = 0; j < n; ++j) v |= (__ldg(row + 32 * w + j) != 0 ? 1u : 0u) << j;
    bits[w] = v;
  }
}

// Adds the weighted value rows of the drafts in `bits`, whose V rows are not
// finite and were left out of the product, to one row's partial O in memory:
// only rows that see such a draft come here (see the draft tile).
template <bool BF16>
__device__ __noinline__ void tree_add_special(const TreeParams& p, int b, int h, int g, int t, uint32_t bits, int j0,
                                              float m, float* o) {
  const uint16_t* q = p.q + b * p.q_sb + (static_cast<int64_t>(h) * p.G + g) * p.q_sh + t * p.q_st;
  for (; bits != 0u; bits &= bits - 1u) {
    const int j = j0 + __ffs(bits) - 1;
    const uint16_t* k = p.k_new + b * p.kn_sb + h * p.kn_sh + j * p.kn_st;
    const uint16_t* v = p.v_new + b * p.vn_sb + h * p.vn_sh + j * p.vn_st;
    float s = 0.f;
    for (int d = 0; d < p.D; ++d) s = fmaf(elem_to_float<BF16>(q[d]), elem_to_float<BF16>(k[d]), s);
    const float w = ex2_approx(s * p.sc - m);
    for (int c = 0; c < p.D; ++c) o[c] += w * elem_to_float<BF16>(v[c]);
  }
}

template <bool BF16>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;
  return (w & E) == E || ((w >> 16) & E) == E;
}

template <bool BF16, int DP, bool DUAL>
__global__ void __launch_bounds__(384, 1)
    fe_tree_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                   const __grid_constant__ CUtensorMap tkn, const __grid_constant__ CUtensorMap tvn,
                   const __grid_constant__ TreeParams p) {
  using C = TreeCfg<DP, DUAL>;
  constexpr int NG = C::NG;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* k_full = q_full + 1;
  uint64_t* v_full = k_full + C::STAGES;
  uint64_t* k_empty = v_full + C::STAGES;
  uint64_t* v_empty = k_empty + C::STAGES;
  uint64_t* s_full = v_empty + C::STAGES;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* drain = o_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  // Drafts whose V row is not finite, 128 bits, one set per segment parity.
  uint32_t* special = tmem_holder + 4;
  int* scratch = reinterpret_cast<int*>(special + 8);

  const int warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_init(q_full, 4 * NG);
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
  // Ends with a block barrier, which also publishes the barriers and TMEM.
  DecWalk walk = dec_walk_init<C::THREADS>(p.lengths, p.B * p.Hkv, p.capacity, p.MT, blockIdx.x, p.nctas, scratch,
                                           blockIdx.x == 0 ? p.base : nullptr);
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const uint64_t TO = p.timeout_ns;
  DecSegment sg;

  if (warp >= 8) {
    setmaxnreg_dec<FWD_REGS_LOW>();
    if (warp == 8) {
      // ---------------------------------------------------------- producer --
      if (lane == 0) {
        tma_prefetch_desc(&tk);
        tma_prefetch_desc(&tv);
        tma_prefetch_desc(&tkn);
        tma_prefetch_desc(&tvn);
        uint32_t loads[C::STAGES];
        for (int s = 0; s < C::STAGES; ++s) loads[s] = 0;
        bool ok = true;
        uint32_t it = 0;
        while (ok && walk.next(sg)) {
          const int b = sg.bh / p.Hkv, h = sg.bh - b * p.Hkv;
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
          auto tile_of = [&](int i) { return it0 + static_cast<uint32_t>(DUAL ? i >> 1 : i); };
          auto issue_s = [&](int i) -> bool {
            const uint32_t tile = tile_of(i);
            const int s = tile % C::STAGES, t = i % NG;
            if (!DUAL || (i & 1) == 0) {
              if (!mbar_wait(&k_full[s], (tile / C::STAGES) & 1, TO, abort_flag)) return false;
              tc_fence_after();
            }
            const uint32_t a = dq_lo + (DUAL ? t * TILE16 : 0u);
            const uint32_t bb = dk_lo + s * TILE16;
#pragma unroll 8
            for (int kk = 0; kk < DP / 16; ++kk) {
              const uint32_t off = static_cast<uint32_t>(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4);
              umma_ss_lohi(tmem + t * 128, a + off, dq_hi, bb + off, dk_hi, ID_S, kk > 0);
            }
            umma_commit(&s_full[t]);
            if (!DUAL || (i & 1) == 1) umma_commit(&k_empty[s]);
            return true;
          };
          ok = mbar_wait(q_full, nseg & 1, TO, abort_flag);
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
          // A group without a step still learns that the segment's products
          // are done (it rewrites its share of the query tile next).
          if (ok && steps < NG) umma_commit(&o_full[1]);
          it0 += ntile;
          ++nseg;
        }
        umma_commit(drain);
        mbar_wait_inflight(drain, 0, TO);
      }
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
      bool ok = true;
      uint32_t it0 = 0, nseg = 0, ns = 0;  // key tiles before, segments, S tiles of this group
      for (; walk.next(sg); ++nseg) {
        const int b = sg.bh / p.Hkv, h = sg.bh - b * p.Hkv;
        const int row = sg.mt * C::ROWS + (DUAL ? t * 128 : 0) + r;  // of the item's G*T queries
        const bool live = row < p.M;
        const bool warp_live = row - static_cast<int>(lane) < p.M;
        const int g = live ? row / p.T : 0, tt = live ? row - g * p.T : 0;
        uint32_t* spec = special + (nseg & 1) * 4;
        // ---- query tile into shared memory (padding rows and channels zero)
        {
          const int rows0 = DUAL ? t * 128 : t * (128 / NG);
          const int nrows = DUAL ? 128 : 128 / NG;
          constexpr int CPR = DP / 8;
          const int tid = r;
          const uint16_t* qb = p.q + b * p.q_sb + static_cast<int64_t>(h) * p.G * p.q_sh;
          for (int i0 = tid; i0 < nrows * CPR; i0 += 128 * 4) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int i = i0 + u * 128;
              v[u] = make_uint4(0u, 0u, 0u, 0u);
              const int qr = sg.mt * C::ROWS + rows0 + i / CPR;
              if (i < nrows * CPR && qr < p.M) {
                const int qg = qr / p.T;
                v[u] = load_row_chunk(qb + qg * p.q_sh + (qr - qg * p.T) * p.q_st, i % CPR, p.D, p.q_vec);
              }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int i = i0 + u * 128;
              if (i < nrows * CPR) {
                const int lr = rows0 + i / CPR;
                *reinterpret_cast<uint4*>(smem + C::OFF_Q + (lr >> 7) * C::TILE +
                                          sw128_offset(lr & 127, i % CPR, 16384)) = v[u];
              }
            }
          }
          if (t == 0 && r < 4) spec[r] = 0u;
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(q_full);
        }
        float m_used = TREE_M0, l = 0.f;
        bool first = true;
        const int ntile = sg.j1 - sg.j0;
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
            uint8_t* vt = smem + C::OFF_V + s * C::TILE + r * 128;
            bool clear = r > lim;
            if (drafts && !clear) {
              bool bad = false;
              for (int c = 0; c < C::NCH; ++c)
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                  const uint4 w = *reinterpret_cast<const uint4*>(vt + c * 16384 + ((u ^ (r & 7)) << 4));
                  bad = bad || not_finite2<BF16>(w.x) || not_finite2<BF16>(w.y) || not_finite2<BF16>(w.z) ||
                        not_finite2<BF16>(w.w);
                }
              if (bad) atomicOr(&spec[r >> 5], 1u << (r & 31));
              clear = bad;
            }
            if (clear) {
              for (int c = 0; c < C::NCH; ++c)
#pragma unroll
                for (int u = 0; u < 8; ++u)
                  *reinterpret_cast<uint4*>(vt + c * 16384 + ((u ^ (r & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
          }
          if (warp_live) {
            float x[128];
            {
              uint32_t* xr = reinterpret_cast<uint32_t*>(x);
              tmem_ld64_sync(tS, xr);
              tmem_ld64_sync(tS + 64, xr + 64);
            }
            uint32_t bits[4] = {0u, 0u, 0u, 0u};
            if (drafts) {
              if (live) tree_bits(p, b, tt, bits);
              tree_softmax_tile<BF16, DP, 2>(x, first, lim, bits, sc, sce, sc_pos, m_used, l, tS, tO);
            } else if (lim < 127) {
              tree_softmax_tile<BF16, DP, 1>(x, first, lim, bits, sc, sce, sc_pos, m_used, l, tS, tO);
            } else {
              tree_softmax_tile<BF16, DP, 0>(x, first, lim, bits, sc, sce, sc_pos, m_used, l, tS, tO);
            }
          }
          first = false;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[t]);
        }
        if (ok) ok = warp_all(mbar_wait(&o_full[t], nseg & 1, TO, abort_flag));
        tc_fence_after();
        // ---- partial result of this run for the row
        const int64_t slot = (static_cast<int64_t>(sg.bh) * p.MT + sg.mt + blockIdx.x) * C::PARTS + (DUAL ? 0 : t);
        const int pr = (DUAL ? t * 128 : 0) + r;
        const float nan = __int_as_float(0x7fffffff);
        if (live) p.stats[slot * p.R + pr] = ok ? make_float2(m_used, l) : make_float2(nan, nan);
        if (ok && !first && warp_live) {
          float* dst = p.acc + (slot * p.R + pr) * p.D4;
#pragma unroll 1
          for (int c0 = 0; c0 < DP; c0 += 32) {
            uint32_t o[32];
            tmem_ld32_sync(tO + c0, o);
            if (live) {
#pragma unroll
              for (int q4 = 0; q4 < 8; ++q4)
                if (c0 + q4 * 4 < p.D4)
                  *reinterpret_cast<uint4*>(dst + c0 + q4 * 4) =
                      make_uint4(o[4 * q4], o[4 * q4 + 1], o[4 * q4 + 2], o[4 * q4 + 3]);
            }
          }
          // Only the group that took the draft tile adds its special rows.
          if ((spec[0] | spec[1] | spec[2] | spec[3]) != 0u && live && (DUAL || (ntile - 1) % NG == t)) {
            uint32_t bits[4];
            tree_bits(p, b, tt, bits);
#pragma unroll
            for (int w = 0; w < 4; ++w) tree_add_special<BF16>(p, b, h, g, tt, bits[w] & spec[w], 32 * w, m_used, dst);
          }
        }
        tc_fence_before();
        it0 += ntile;
      }
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

constexpr int TREE_JOIN_THREADS = 128;

// Joins the runs' partials of one query row (one warp): the rows' weights
// 2^(m_i - max m) in the order of the runs.
template <bool BF16>
__global__ void __launch_bounds__(TREE_JOIN_THREADS) fe_tree_join_kernel(const __grid_constant__ TreeParams p, int parts, int rows_per_item) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t orow = static_cast<int64_t>(blockIdx.x) * (TREE_JOIN_THREADS / 32) + (threadIdx.x >> 5);
  if (orow >= static_cast<int64_t>(p.B) * p.Hkv * p.M) return;
  const int bh = static_cast<int>(orow / p.M);
  const int row = static_cast<int>(orow - static_cast<int64_t>(bh) * p.M);
  const int mt = row / rows_per_item, pr = row - mt * rows_per_item;
  const int total = p.base[p.B * p.Hkv];
  const int per = (total + p.nctas - 1) / p.nctas;
  const int start = p.base[bh];
  const int tiles = (p.base[bh + 1] - start) / p.MT;
  const int u0 = start + mt * tiles;
  const int c0 = u0 / per, c1 = (u0 + tiles - 1) / per;
  const int64_t slot0 = (static_cast<int64_t>(bh) * p.MT + mt + c0) * parts;
  const int n = (c1 - c0 + 1) * parts;
  float m = TREE_M0, bad = 0.f;
  for (int i = lane; i < n; i += 32) {
    const float2 st = p.stats[(slot0 + i) * p.R + pr];
    if (st.y != 0.f) m = fmaxf(m, st.x);
    bad += st.x * 0.f + st.y * 0.f;  // NaN or inf statistics mark the row
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    bad += __shfl_xor_sync(0xffffffffu, bad, o);
  }
  // lane holds columns 4*lane .. +3, and the same 128 further on
  float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  float l = 0.f;
  for (int i0 = 0; i0 < n; i0 += 32) {
    float2 st = make_float2(TREE_M0, 0.f);
    if (i0 + lane < n) st = p.stats[(slot0 + i0 + lane) * p.R + pr];
    const float w_mine = st.y != 0.f ? exp2f(st.x - m) : 0.f;
    const float l_mine = st.y;
    const int k = min(32, n - i0);
#pragma unroll 4
    for (int i = 0; i < k; ++i) {
      const float w = __shfl_sync(0xffffffffu, w_mine, i);
      const float li = __shfl_sync(0xffffffffu, l_mine, i);
      if (li == 0.f) continue;  // this run saw no key of the row
      l = fmaf(w, li, l);
      const float* src = p.acc + ((slot0 + i0 + i) * p.R + pr) * p.D4;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = e * 128 + lane * 4;
        if (c < p.D4) {
          const float4 v = *reinterpret_cast<const float4*>(src + c);
          acc[e][0] = fmaf(w, v.x, acc[e][0]);
          acc[e][1] = fmaf(w, v.y, acc[e][1]);
          acc[e][2] = fmaf(w, v.z, acc[e][2]);
          acc[e][3] = fmaf(w, v.w, acc[e][3]);
        }
      }
    }
  }
  l += bad;
  const bool none = l == 0.f;
  const float inv = none ? 0.f : 1.0f / l;
  uint16_t* out = p.out + orow * p.D;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int c = e * 128 + lane * 4;
    if (c >= p.D) continue;
    const uint32_t a = pack2<BF16>(acc[e][0] * inv, acc[e][1] * inv);
    const uint32_t b2 = pack2<BF16>(acc[e][2] * inv, acc[e][3] * inv);
    if ((p.D & 3) == 0) {
      *reinterpret_cast<uint2*>(out + c) = make_uint2(a, b2);
    } else {
      const uint16_t w[4] = {static_cast<uint16_t>(a), static_cast<uint16_t>(a >> 16), static_cast<uint16_t>(b2),
                             static_cast<uint16_t>(b2 >> 16)};
      for (int i = 0; i < 4 && c + i < p.D; ++i) out[c + i] = w[i];
    }
  }
  if (lane == 0) p.lse[orow] = none ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

}  // namespace fe
