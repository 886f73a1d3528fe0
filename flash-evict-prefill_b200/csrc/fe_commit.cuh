// Commit of accepted drafts: their attention weight onto every cached token,
// and their K/V rows onto the end of the cache (sm_100a).
//
// With the accepted drafts a_0..a_{n-1} of a sequence (in order) and the row
// sums lse of their attention,
//   w_i     = exp(-decay * (n-1-i))
//   mass_k <- exp(-decay * n) * mass_k + norm_k * sum_{i,g} w_i exp(scale*q_{i,g}.k - lse_{i,g})
// for cached tokens, the same sum over the accepted drafts that see it for each
// appended token -- the importance of the prefill's replay, continued: the
// weights are those it would give with the new tokens at the end.
//
// fe_commit_mass_kernel is key-stationary like the replay: S^T = K Q^T with the
// 128 keys of a tile on the TMEM lanes and the accepted queries (n*G rows,
// gathered and padded to 16) as columns, so each thread owns one key and sums
// its row in registers: no shuffles, no atomics, one FP32 store per key.  What
// bounds it is reading K once (2*D bytes a token).  The normaliser and weight
// fold into one exponent bias per column: w exp(s - lse) = exp2(x*sc - bias).
//
// Work is split over the SMs as in fe_decode.cuh, the last tile of a row being
// its drafts.  Four warpgroups take every fourth tile of a run, each with its
// own 128-column S^T buffer; one warp streams K tiles by TMA, one issues the
// products.  The queries of a run stay in shared memory; more than ROWS of
// them take further launches.  Two more warps append the accepted rows of the
// runs that end a row, and wait only for the new tokens' weights.  (In the
// warpgroup that sums them the appending cost the loop over the tiles its
// registers: 33 -> 43 us for the batch of 16.)  Every CTA reads the lengths, so in place they are
// written by the last CTA to finish (a counter in the cache, back at zero then).
#pragma once

#include "fe_decode.cuh"

namespace fe {

constexpr int COMMIT_MAX_ACCEPTED = 128;

struct CommitParams {
  const uint16_t* q;
  int64_t q_sb, q_sh, q_st;
  const float* lse;         // [B, Hq, T]
  const int32_t* accepted;  // [B, A], negative: none
  const uint8_t* tree;
  int64_t tree_sb;
  const int32_t* lengths;
  const float* mass_in;
  const float* norms_in;    // or null
  const int32_t* pos_in;
  float* mass_out;
  float* norms_out;
  int32_t* pos_out;
  float* new_mass;       // workspace [B*Hkv, T]: weight of each draft so far, between launches
  int32_t* new_lengths;  // [B*Hkv]: the output lengths, or (in place) workspace
  int32_t* len_out;      // in place: the lengths, written by the last CTA
  int32_t* sync;         // in place: CTAs that are done, 0 between launches
  const uint16_t* k_new;
  int64_t kn_sb, kn_sh, kn_st;
  const uint16_t* v_new;
  int64_t vn_sb, vn_sh, vn_st;
  uint16_t* k;
  int64_t k_sb, k_sh, k_st;
  uint16_t* v;
  int64_t v_sb, v_sh, v_st;
  const int32_t* new_positions;  // [B, T]
  int B, Hq, Hkv, G, T, A, D, capacity, nctas;
  int extra;           // key tiles that beginning a row costs
  int row0;            // first query row (i*G + g) of this launch
  int last;            // the last launch: append
  int copy;            // mass_out, norms_out, pos_out are other buffers: fill them
  int rows_vec;        // K/V rows can be moved 16 bytes at a time
  float sc;            // scale * log2(e)
  double decay_log2;
  int q_vec, tree_vec; // query rows, mask rows can be read 16 bytes at a time
  uint64_t timeout_ns;
};

// Registers: launched at 96 a thread (640 threads); the control warpgroup drops
// to 64 and the four that reduce rise to 104 (4*128*104 + 128*64 = 640*96).
constexpr uint32_t COMMIT_REGS_HIGH = 104, COMMIT_REGS_LOW = 64;
constexpr int COMMIT_REGS_NEEDED = (4 * 128 * 104 + 128 * 64) / 640;

template <int DP>
struct CommitCfg {
  static constexpr int WGS = 4;
  static constexpr int ROWS = DP <= 128 ? 256 : 128;  // query rows per launch
  static constexpr int TILE = 128 * DP * 2;
  static constexpr int NCH = DP / 64;
  static constexpr int QTILES = ROWS / 128;
  static constexpr int STAGES = DP <= 64 ? 8 : (DP <= 128 ? 4 : 2);
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = QTILES * TILE;
  static constexpr int OFF_BIAS = OFF_K + STAGES * TILE;
  static constexpr int OFF_MASK = OFF_BIAS + ROWS * 4;                       // uint32[128][4]
  static constexpr int OFF_LIST = OFF_MASK + COMMIT_MAX_ACCEPTED * 16;      // int[128]
  static constexpr int OFF_COL = OFF_LIST + COMMIT_MAX_ACCEPTED * 4;        // uint32[4][ROWS]: masks by column
  static constexpr int OFF_NEW = OFF_COL + ROWS * 16;                       // float[2][128]: weights of new tokens
  static constexpr int OFF_APP = OFF_NEW + 2 * 128 * 4;                     // int list[128], float norm[128]
  static constexpr int OFF_BAR = OFF_APP + COMMIT_MAX_ACCEPTED * 8;
  // q_full, k_full[S], k_empty[S], s_full[WGS], s_free[WGS], drain, new_full[2], new_empty[2]
  static constexpr int NBAR = 1 + 2 * STAGES + 2 * WGS + 1 + 4;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int SMEM = OFF_MISC + 16 + DEC_SCRATCH_INTS * 4 + 1024;
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  static constexpr int PRODUCER = WGS * 4;
  static constexpr int ISSUER = WGS * 4 + 1;
  static constexpr int APPEND = WGS * 4 + 2;  // two warps
  static constexpr int THREADS = (WGS * 4 + 4) * 32;
};

// Number of accepted drafts of sequence b, by one converged warp; with list !=
// nullptr their draft indices in order are written there.
__device__ __forceinline__ int accepted_drafts(const int32_t* accepted, int A, int T, int b, int* list) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int a0 = 0; a0 < A; a0 += 32) {
    const int j = a0 + lane < A ? accepted[static_cast<int64_t>(b) * A + a0 + lane] : -1;
    const bool valid = j >= 0 && j < T;
    const uint32_t bal = __ballot_sync(0xffffffffu, valid);
    if (valid && list != nullptr) list[n + __popc(bal & ((1u << lane) - 1u))] = j;
    n += __popc(bal);
  }
  return n;
}

// Sum over `cols` (a multiple of 16, at most 128 / PARTS) query columns of one key's
// S^T row of exp2(x * sc + bias); `release` is called once the row has been
// read.  FULL: 128 columns, unrolled.  DRAFT: only columns with bit `bit` of their word in
// `masks` set.
template <int PARTS, bool FULL, bool DRAFT, typename Release>
__device__ __forceinline__ float commit_reduce(uint32_t tS, int cols, float sc, const float* bias, const uint32_t* masks,
                                               int bit, Release release) {
  const uint64_t sc2 = f2_pack(sc, sc);
  uint64_t acc2[4] = {0ull, 0ull, 0ull, 0ull};
  auto chunk = [&](int c0, const float (&x)[16]) {
#pragma unroll
    for (int c4 = 0; c4 < 16; c4 += 4) {
      const float4 nb = *reinterpret_cast<const float4*>(bias + c0 + c4);
      uint4 see = make_uint4(0u, 0u, 0u, 0u);
      if (DRAFT) see = *reinterpret_cast<const uint4*>(masks + c0 + c4);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = c4 + 2 * u;
        const uint64_t a2 = f2_fma(f2_pack(x[c], x[c + 1]), sc2, u == 0 ? f2_pack(nb.x, nb.y) : f2_pack(nb.z, nb.w));
        float a0, a1;
        f2_unpack(a2, a0, a1);
        if (DRAFT) {
          a0 = (((u == 0 ? see.x : see.z) >> bit) & 1u) ? a0 : -INFINITY;
          a1 = (((u == 0 ? see.y : see.w) >> bit) & 1u) ? a1 : -INFINITY;
        }
        acc2[(c >> 1) & 3] = f2_add(acc2[(c >> 1) & 3], f2_pack(ex2_approx(a0), ex2_approx(a1)));
      }
    }
  };
  if constexpr (PARTS > 1) {
#pragma unroll 1
    for (int c0 = 0; c0 < cols; c0 += 16) {
      float x[16], y[16];
      // (Two parts at a time: all four at once would not fit the registers.)
#pragma unroll
      for (int i = 0; i < PARTS; i += 2) {
        float z[16];
        tmem_ld16_nowait(tS + i * (128 / PARTS) + c0, reinterpret_cast<uint32_t*>(y));
        tmem_ld16_nowait(tS + (i + 1) * (128 / PARTS) + c0, reinterpret_cast<uint32_t*>(z));
        tmem_wait_ld16(reinterpret_cast<uint32_t*>(y));
        tmem_wait_ld16(reinterpret_cast<uint32_t*>(z));
#pragma unroll
        for (int c = 0; c < 16; ++c) x[c] = i == 0 ? y[c] + z[c] : x[c] + (y[c] + z[c]);
      }
      if (c0 + 16 >= cols) release();
      chunk(c0, x);
    }
  } else {
    // The next 16 columns are in flight while these are summed.
    float xa[16], xb[16];
    tmem_ld16_nowait(tS, reinterpret_cast<uint32_t*>(xa));
    tmem_wait_ld16(reinterpret_cast<uint32_t*>(xa));
    auto pair = [&](int c0, bool more_b, bool more_a) {
      if (more_b) tmem_ld16_nowait(tS + c0 + 16, reinterpret_cast<uint32_t*>(xb));
      else release();
      chunk(c0, xa);
      if (!more_b) return;
      tmem_wait_ld16(reinterpret_cast<uint32_t*>(xb));
      if (more_a) tmem_ld16_nowait(tS + c0 + 32, reinterpret_cast<uint32_t*>(xa));
      else release();
      chunk(c0 + 16, xb);
      if (more_a) tmem_wait_ld16(reinterpret_cast<uint32_t*>(xa));
    };
    if (FULL) {
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 32) pair(c0, true, c0 < 96);
    } else {
#pragma unroll 1
      for (int c0 = 0; c0 < cols; c0 += 32) pair(c0, c0 + 16 < cols, c0 + 32 < cols);
    }
  }
  float s[8];
#pragma unroll
  for (int u = 0; u < 4; ++u) f2_unpack(acc2[u], s[2 * u], s[2 * u + 1]);
  return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// Appends the K/V rows of cache row bh's accepted drafts, with their norms and
// positions, by two warps (64 threads), four rows a warp in flight.  The norms
// are left in shared memory for the weights that follow.
template <bool BF16>
__device__ __forceinline__ void commit_append_rows(const CommitParams& p, int bh, int b, int h, int len, int fit,
                                                   const int* list, float* norms, int warp, int lane) {
  constexpr int U = 4;
  const int64_t base = static_cast<int64_t>(bh) * p.capacity;
  const uint16_t* kn = p.k_new + b * p.kn_sb + h * p.kn_sh;
  const uint16_t* vn = p.v_new + b * p.vn_sb + h * p.vn_sh;
  uint16_t* kc = p.k + b * p.k_sb + h * p.k_sh;
  uint16_t* vc = p.v + b * p.v_sb + h * p.v_sh;
  for (int i0 = warp * U; i0 < fit; i0 += 2 * U) {
    const int count = min(U, fit - i0);
    float norm[U];
#pragma unroll
    for (int u = 0; u < U; ++u) norm[u] = 0.f;
    if (p.rows_vec) {
      const int cpr = p.D / 8;
      for (int c = lane; c < 2 * cpr; c += 32) {
        const bool is_v = c >= cpr;
        const int o = (is_v ? c - cpr : c) * 8;
        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = list[i0 + min(u, count - 1)];
          x[u] = *reinterpret_cast<const uint4*>((is_v ? vn + j * p.vn_st : kn + j * p.kn_st) + o);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t slot = len + i0 + u;
          if (u < count) *reinterpret_cast<uint4*>((is_v ? vc + slot * p.v_st : kc + slot * p.k_st) + o) = x[u];
          if (is_v) {
            const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              norm[u] += fabsf(elem_to_float<BF16>(static_cast<uint16_t>(w[e]))) +
                         fabsf(elem_to_float<BF16>(static_cast<uint16_t>(w[e] >> 16)));
          }
        }
      }
    } else {
      for (int c = lane; c < p.D; c += 32)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u >= count) continue;
          const int64_t slot = len + i0 + u;
          const int j = list[i0 + u];
          kc[slot * p.k_st + c] = kn[j * p.kn_st + c];
          const uint16_t e = vn[j * p.vn_st + c];
          vc[slot * p.v_st + c] = e;
          norm[u] += fabsf(elem_to_float<BF16>(e));
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) norm[u] += __shfl_xor_sync(0xffffffffu, norm[u], o);
      if (lane == u && u < count) {
        const int64_t at = base + len + i0 + u;
        if (p.norms_out != nullptr) p.norms_out[at] = norm[u];
        norms[i0 + u] = p.norms_out != nullptr ? norm[u] : 1.0f;
        p.pos_out[at] = p.new_positions[static_cast<int64_t>(b) * p.T + list[i0 + u]];
      }
    }
  }
}

// PARTS: accumulators that a score is summed from, each over a part of the channels
// and 128 / PARTS columns from the next.  The tensor core cuts its FP32 sums off
// where an addition would round them, once every 16 channels, so a score leans
// towards zero, and with it the weights of heavy keys (256 channels in one sum: up to
// 3.4e-6 off where an FP32 product's are 6e-7); the parts are added in FP32 as usual.
template <bool BF16, int DP, int PARTS>
__global__ void __launch_bounds__(CommitCfg<DP>::THREADS, 1)
    fe_commit_mass_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tkn,
                          const __grid_constant__ CommitParams p) {
  using C = CommitCfg<DP>;
  constexpr int CHUNK = 128 / PARTS;  // query columns of a product
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sbias = reinterpret_cast<float*>(smem + C::OFF_BIAS);
  uint32_t* smask = reinterpret_cast<uint32_t*>(smem + C::OFF_MASK);
  int* slist = reinterpret_cast<int*>(smem + C::OFF_LIST);
  uint32_t* scol = reinterpret_cast<uint32_t*>(smem + C::OFF_COL);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + C::STAGES;
  uint64_t* s_full = k_empty + C::STAGES;
  uint64_t* s_free = s_full + C::WGS;
  uint64_t* drain = s_free + C::WGS;
  uint64_t* new_full = drain + 1;
  uint64_t* new_empty = new_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  float* sfade = reinterpret_cast<float*>(tmem_holder + 2);
  int* scratch = reinterpret_cast<int*>(tmem_holder + 4);

  const int warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == C::PRODUCER * 32) {
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tkn);
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    mbar_init(q_full, C::WGS * 4);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int w = 0; w < C::WGS; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&s_free[w], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&new_full[i], 4);
      mbar_init(&new_empty[i], 2);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  if (warp == C::ISSUER) {
    __syncwarp();
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  pdl_wait();  // nothing above reads or writes memory
  DecWalk walk = dec_walk_init<C::THREADS>(p.lengths, p.B * p.Hkv, p.capacity, 1, p.extra, blockIdx.x, p.nctas,
                                               scratch);
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const uint64_t TO = p.timeout_ns;
  DecSegment sg;
  auto rows_of = [&](int b, int n) { return min(max(n * p.G - p.row0, 0), C::ROWS); };

  if (warp >= C::PRODUCER) {
  setmaxnreg_dec<COMMIT_REGS_LOW>();
  if (warp == C::PRODUCER) {
    // ------------------------------------------------------------ producer --
    uint32_t it = 0;
    bool ok = true;
    while (ok && walk.next(sg)) {
      const int b = sg.bh / p.Hkv, h = sg.bh - b * p.Hkv;
      if (rows_of(b, accepted_drafts(p.accepted, p.A, p.T, b, nullptr)) == 0) continue;
      for (int j = sg.j0; j < sg.j1; ++j) {
        if (lane == 0) {
          const int s = it % C::STAGES;
          const uint32_t use = it / C::STAGES;
          const bool drafts = j == sg.tiles - 1;
          if (use > 0) ok = mbar_wait(&k_empty[s], (use - 1) & 1, TO, abort_flag);
          if (ok) {
            mbar_expect_tx(&k_full[s], C::TILE);
            for (int c = 0; c < C::NCH; ++c)
              tma_load_4d(smem + C::OFF_K + s * C::TILE + c * 16384, drafts ? &tkn : &tk, &k_full[s], c * 64,
                          drafts ? 0 : j * DEC_TILE, h, b);
          }
        }
        ok = warp_all(ok);
        if (!ok) break;
        ++it;
      }
    }
    // Every load must have landed before the CTA exits.
    if (lane == 0)
      for (uint32_t i = it > C::STAGES ? it - C::STAGES : 0; i < it; ++i)
        mbar_wait_inflight(&k_full[i % C::STAGES], (i / C::STAGES) & 1, TO);
  } else if (warp == C::ISSUER) {
    // ---------------------------------------------------------- MMA issuer --
    const uint64_t dk = smem_desc_sw128(smem_u32(smem + C::OFF_K), 16, 1024);
    const uint64_t dq = smem_desc_sw128(smem_u32(smem + C::OFF_Q), 16, 1024);
    const uint32_t dk_lo = static_cast<uint32_t>(dk), dk_hi = static_cast<uint32_t>(dk >> 32);
    const uint32_t dq_lo = static_cast<uint32_t>(dq), dq_hi = static_cast<uint32_t>(dq >> 32);
    uint32_t it0 = 0, nq = 0;
    uint32_t began = 0, parity = 0;  // per warpgroup: has had a product; number of them, mod 2
    bool ok = true;
    while (ok && walk.next(sg)) {
      const int b = sg.bh / p.Hkv;
      const int rows = rows_of(b, accepted_drafts(p.accepted, p.A, p.T, b, nullptr));
      if (rows == 0) continue;
      const int ntile = sg.j1 - sg.j0;
      if (lane == 0) {
        ok = mbar_wait(q_full, nq & 1, TO, abort_flag);
        tc_fence_after();
        constexpr int STEPS = DP / 16 / PARTS;  // of 16 channels a part
        const int nch = (rows + CHUNK - 1) / CHUNK;
        // Rounds of a tile per warpgroup, no more than there are stages: they are
        // kept through the chunks of queries, which are inside.
        constexpr int ROUND = C::STAGES < C::WGS ? C::STAGES : C::WGS;
        for (int i0 = 0; i0 < ntile && ok; i0 += ROUND)
          for (int c = 0; c < nch && ok; ++c) {
            const int cols = (min(rows - c * CHUNK, CHUNK) + 15) & ~15;
            const uint32_t id = idesc_f16(128, cols, BF16, false);
#pragma unroll
            for (int u = 0; u < ROUND; ++u) {
              if (i0 + u >= ntile || !ok) continue;
              const int w = (i0 + u) % C::WGS;
              const uint32_t tile = it0 + i0 + u;
              const int s = tile % C::STAGES;
              if (c == 0) ok = mbar_wait(&k_full[s], (tile / C::STAGES) & 1, TO, abort_flag);
              if (ok && ((began >> w) & 1u)) ok = mbar_wait(&s_free[w], ((parity >> w) & 1u) ^ 1u, TO, abort_flag);
              if (!ok) continue;
              began |= 1u << w;
              parity ^= 1u << w;
              tc_fence_after();
              const uint32_t ka = dk_lo + static_cast<uint32_t>(s * (C::TILE >> 4));
              const int row = c * CHUNK;
              const uint32_t qa = dq_lo + static_cast<uint32_t>((row >> 7) * (C::TILE >> 4) + (row & 127) * (128 >> 4));
#pragma unroll
              for (int kk = 0; kk < DP / 16; ++kk) {
                const uint32_t off = static_cast<uint32_t>(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4);
                umma_ss_lohi(tmem + w * 128 + kk / STEPS * CHUNK, ka + off, dk_hi, qa + off, dq_hi, id, kk % STEPS != 0);
              }
              umma_commit(&s_full[w]);
              if (c == nch - 1) umma_commit(&k_empty[s]);
            }
          }
      }
      ok = warp_all(ok);
      it0 += ntile;
      ++nq;
    }
    if (lane == 0) {
      umma_commit(drain);
      mbar_wait_inflight(drain, 0, TO);
    }
  } else {
    // -------------------------------------------------------------- append --
    const int w = warp - C::APPEND;
    int* list = reinterpret_cast<int*>(smem + C::OFF_APP);
    float* norms = reinterpret_cast<float*>(list + COMMIT_MAX_ACCEPTED);
    uint32_t nrow = 0;  // rows whose draft tile this run had
    bool ok = true;
    while (p.last && walk.next(sg)) {
      if (sg.j1 != sg.tiles) continue;
      const int b = sg.bh / p.Hkv, h = sg.bh - b * p.Hkv;
      named_bar_sync(2, 64);  // both warps are done with the previous row's list
      const int n = accepted_drafts(p.accepted, p.A, p.T, b, w == 0 ? list : nullptr);
      named_bar_sync(2, 64);
      const int fit = min(n, p.capacity - sg.len);
      commit_append_rows<BF16>(p, sg.bh, b, h, sg.len, fit, list, norms, w, static_cast<int>(lane));
      named_bar_sync(2, 64);
      if (ok) ok = warp_all(mbar_wait(&new_full[nrow & 1], (nrow >> 1) & 1, TO, abort_flag));
      const float* fresh = reinterpret_cast<const float*>(smem + C::OFF_NEW) + (nrow & 1) * 128;
      for (int i = w * 32 + static_cast<int>(lane); i < fit; i += 64)
        p.mass_out[static_cast<int64_t>(sg.bh) * p.capacity + sg.len + i] =
            ok ? norms[i] * fresh[list[i]] : __int_as_float(0x7fffffff);
      __syncwarp();
      if (lane == 0) mbar_arrive(&new_empty[nrow & 1]);
      ++nrow;
      if (w == 0) {
        bool bad = false;
        if (h == 0)
          for (int a = lane; a < p.A; a += 32) bad = bad || p.accepted[static_cast<int64_t>(b) * p.A + a] >= p.T;
        if (bad) raise_status(FE_STATUS_BAD_INDEX);
        if (lane == 0) {
          p.new_lengths[sg.bh] = sg.len + fit;
          if (fit < n) raise_status(FE_STATUS_CACHE_FULL);
        }
      }
    }
  }
  } else {
    setmaxnreg_inc<COMMIT_REGS_HIGH>();
    // ------------------------------------------------ reduce (thread = key) --
    const int wg = warp >> 2;
    const int kr = ((warp & 3) << 5) + static_cast<int>(lane);
    const uint32_t tS = tmem + (static_cast<uint32_t>((warp & 3) << 5) << 16) + wg * 128;
    const int tid = threadIdx.x;
    constexpr int RT = C::WGS * 128;
    uint32_t li = 0, nrow = 0;  // S^T tiles of this warpgroup; rows whose draft tile the run had
    bool ok = true;
    for (; walk.next(sg); nrow += sg.j1 == sg.tiles) {
      const int b = sg.bh / p.Hkv, h = sg.bh - b * p.Hkv;
      // Everyone is done with the previous run's queries (every product that
      // read them has been waited for by the warpgroup it fed).
      named_bar_sync(1, RT);
      const int n = accepted_drafts(p.accepted, p.A, p.T, b, warp == 0 ? slist : nullptr);
      const int rows = rows_of(b, n);
      const int ntile = sg.j1 - sg.j0;
      const int i_first = p.row0 / p.G;
      if (tid == 0) *sfade = p.row0 == 0 ? static_cast<float>(exp2(-p.decay_log2 * n)) : 1.0f;
      named_bar_sync(1, RT);
      const float fade = *sfade;
      if (rows > 0) {
        // Three warpgroups gather the queries while the fourth makes the biases
        // and masks: one memory latency instead of three.
        constexpr int QT = (C::WGS - 1) * 128;
        const int padded = (rows + 15) & ~15;
        constexpr int CPR = DP / 8;
        const uint16_t* qb = p.q + b * p.q_sb + static_cast<int64_t>(h) * p.G * p.q_sh;
        for (int i = tid; wg < C::WGS - 1 && i < padded * CPR; i += QT) {
          const int r = i / CPR, chunk = i % CPR;
          uint8_t* dst = smem + C::OFF_Q + (r >> 7) * C::TILE + sw128_offset(r & 127, chunk, 16384);
          // (Padding repeats the launch's first query: a score of zeros would be NaN
          // for a key that is not finite, where that query's may be -inf and add 0.)
          const int row = p.row0 + (r < rows ? r : 0), qi = row / p.G, g = row - qi * p.G;
          const uint16_t* src = qb + g * p.q_sh + slist[qi] * p.q_st;
          if (p.q_vec) {
            const bool live = chunk * 8 < p.D;
            cp_async16(dst, live ? src + chunk * 8 : qb, live);
          } else {
            *reinterpret_cast<uint4*>(dst) = load_row_chunk(src, chunk, p.D);
          }
        }
        for (int r = tid - QT; wg == C::WGS - 1 && r < padded; r += 128) {
          float bias = -INFINITY;  // padding, and rows that saw nothing, add 0
          if (r < rows) {
            const int qi = (p.row0 + r) / p.G, g = p.row0 + r - qi * p.G;
            const float lse = p.lse[(static_cast<int64_t>(b) * p.Hq + h * p.G + g) * p.T + slist[qi]];
            // Formed in 64 bits and rounded once: the rounding of its two terms
            // would be up to 1e-6 of a weight each.
            if (lse != -INFINITY)
              bias = static_cast<float>(-(p.decay_log2 * (n - 1 - qi) + static_cast<double>(lse) * 1.4426950408889634));
          }
          sbias[r] = bias;
        }
        if (wg == C::WGS - 1 && sg.j1 == sg.tiles) {
          // Which drafts each accepted query of this launch sees, then by column.
          const int nq = (p.row0 + rows - 1) / p.G - i_first + 1;
          for (int i = tid - QT; i < nq * 4; i += 128) {
            const int t = slist[i_first + (i >> 2)], w = i & 3;
            const int cnt = min(max((p.tree == nullptr ? t + 1 : p.T) - 32 * w, 0), 32);
            smask[i] = p.tree == nullptr ? low_bits(cnt)
                                         : mask_word(p.tree + b * p.tree_sb + static_cast<int64_t>(t) * p.T + 32 * w, cnt, p.tree_vec);
          }
          named_bar_sync(3, 128);
          for (int r = tid - QT; r < padded; r += 128) {
            const int i = r < rows ? (p.row0 + r) / p.G - i_first : 0;
            const uint4 m = *reinterpret_cast<const uint4*>(smask + i * 4);
            scol[r] = m.x;
            scol[C::ROWS + r] = m.y;
            scol[2 * C::ROWS + r] = m.z;
            scol[3 * C::ROWS + r] = m.w;
          }
        }
        cp_async_wait_all();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        named_bar_sync(1, RT);
      }
      const int nch = (rows + CHUNK - 1) / CHUNK;
      for (int i = wg; i < ntile; i += C::WGS) {
        const int j = sg.j0 + i;
        const bool drafts = j == sg.tiles - 1;
        const int slot = j * DEC_TILE + kr;
        const bool live = drafts ? kr < p.T : slot < sg.len;
        const int64_t at = static_cast<int64_t>(sg.bh) * p.capacity + slot;
        const int64_t at_new = static_cast<int64_t>(sg.bh) * p.T + kr;
        float mass = 0.f, norm = 1.f;
        if (live && !drafts) {
          mass = p.row0 == 0 ? p.mass_in[at] : p.mass_out[at];
          if (p.norms_in != nullptr) norm = p.norms_in[at];
          if (p.copy && p.row0 == 0) {
            p.pos_out[at] = p.pos_in[at];
            if (p.norms_out != nullptr) p.norms_out[at] = norm;
          }
        } else if (live && p.row0 > 0) {
          mass = p.new_mass[at_new];
        }
        float total = 0.f;
        for (int c = 0; c < nch && ok; ++c) {
          ok = warp_all(mbar_wait(&s_full[wg], li & 1, TO, abort_flag));
          if (!ok) break;
          ++li;
          tc_fence_after();
          const int cols = (min(rows - c * CHUNK, CHUNK) + 15) & ~15;
          auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[wg]);
          };
          const float* bias = sbias + c * CHUNK;
          if (drafts)
            total += commit_reduce<PARTS, false, true>(tS, cols, p.sc, bias, scol + (kr >> 5) * C::ROWS + c * CHUNK, kr & 31, release);
          else if (PARTS == 1 && cols == 128)
            total += commit_reduce<PARTS, true, false>(tS, cols, p.sc, bias, nullptr, 0, release);
          else
            total += commit_reduce<PARTS, false, false>(tS, cols, p.sc, bias, nullptr, 0, release);
        }
        // Aborted (watchdog): the sum is incomplete; store NaN.
        if (!ok) total = __int_as_float(0x7fffffff);
        if (live && !drafts) p.mass_out[at] = fmaf(norm, total, mass * fade);
        if (drafts && p.last) {
          // Hand the new tokens' weights to the appending warps.
          if (nrow >= 2 && ok) ok = warp_all(mbar_wait(&new_empty[nrow & 1], ((nrow >> 1) - 1) & 1, TO, abort_flag));
          reinterpret_cast<float*>(smem + C::OFF_NEW)[(nrow & 1) * 128 + kr] = mass + total;
          __syncwarp();
          if (lane == 0) mbar_arrive(&new_full[nrow & 1]);
        } else if (drafts && live) {
          p.new_mass[at_new] = mass + total;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::ISSUER) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (p.last && !p.copy) {
    // In place: everyone has read the lengths once every CTA has come here.
    if (threadIdx.x == 0) {
      __threadfence();
      scratch[0] = atomicAdd(p.sync, 1) == static_cast<int>(gridDim.x) - 1;
      __threadfence();
    }
    __syncthreads();
    if (scratch[0]) {
      for (int i = threadIdx.x; i < p.B * p.Hkv; i += C::THREADS) p.len_out[i] = __ldcg(p.new_lengths + i);
      if (threadIdx.x == 0) *p.sync = 0;
    }
  }
}

}  // namespace fe
