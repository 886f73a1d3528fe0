// Host side of the decode entry points (included by fe_api.cu, whose checks,
// tensor maps and error reporting it uses).
#pragma once

namespace {

// Limits of the decode kernels: a tree's drafts are one key tile, and the query
// heads of a KV head with one draft are at most two query tiles.
constexpr int64_t kMaxDrafts = 128;
constexpr int64_t kMaxGroup = 256;

int sm_count(int dev) {
  static std::atomic<int> cached[kMaxDevices];
  if (dev < 0 || dev >= kMaxDevices) return 148;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

int check_cache(const fe_cache* c) {
  if (!c) return fail(FE_STATUS_INVALID, "null cache");
  if (c->batch < 1 || c->kv_heads < 1 || c->capacity < 1 || c->channels < 1)
    return fail(FE_STATUS_INVALID, "empty cache: batch=%lld kv_heads=%lld capacity=%lld channels=%lld",
                (long long)c->batch, (long long)c->kv_heads, (long long)c->capacity, (long long)c->channels);
  if (c->dtype != FE_DTYPE_F16 && c->dtype != FE_DTYPE_BF16) return fail(FE_STATUS_INVALID, "dtype must be f16 or bf16");
  if (c->channels > 256) return fail(FE_STATUS_INVALID, "channels must be <= 256");
  if (c->capacity > (int64_t(1) << 30) || c->batch * c->kv_heads > (int64_t(1) << 24))
    return fail(FE_STATUS_UNSUPPORTED, "cache too large");
  if (!c->k || !c->v || !c->lengths) return fail(FE_STATUS_INVALID, "null pointer");
  return FE_STATUS_OK;
}

// The layout fields of a cache (everything the tensor maps depend on).
uint64_t layout_hash(const fe_cache* c) {
  const uint64_t f[] = {reinterpret_cast<uint64_t>(c->k), reinterpret_cast<uint64_t>(c->v), (uint64_t)c->k_strides[0],
                        (uint64_t)c->k_strides[1], (uint64_t)c->k_strides[2], (uint64_t)c->k_strides[3],
                        (uint64_t)c->v_strides[0], (uint64_t)c->v_strides[1], (uint64_t)c->v_strides[2],
                        (uint64_t)c->v_strides[3], (uint64_t)c->batch, (uint64_t)c->kv_heads, (uint64_t)c->capacity,
                        (uint64_t)c->channels, (uint64_t)c->dtype};
  uint64_t h = 1469598103934665603ull;
  for (uint64_t x : f) h = (h ^ x) * 1099511628211ull ^ (h >> 29);
  return h | 1;  // 0 marks maps that were never made
}

// The cache's tensor maps: those that fe_cache_prepare left in it, as long as
// they are of this layout, else made here.  tv may be null.
int cache_maps(const fe_cache* c, CUtensorMap* tk, CUtensorMap* tv) {
  static_assert(sizeof(CUtensorMap) == sizeof(c->map_k), "a tensor map is 128 bytes");
  if (c->maps_of != 0 && c->maps_of == layout_hash(c)) {
    memcpy(tk, c->map_k, sizeof(*tk));
    if (tv) memcpy(tv, c->map_v, sizeof(*tv));
    return FE_STATUS_OK;
  }
  int rc = make_map(tk, c->k, c->k_strides, c->batch, c->kv_heads, c->capacity, c->channels, c->dtype, "cache k");
  if (rc || !tv) return rc;
  return make_map(tv, c->v, c->v_strides, c->batch, c->kv_heads, c->capacity, c->channels, c->dtype, "cache v");
}

int check_drafts(const fe_cache* c, int64_t q_heads, int64_t drafts) {
  if (q_heads < 1 || q_heads % c->kv_heads) return fail(FE_STATUS_INVALID, "q_heads must be divisible by kv_heads");
  if (drafts < 1) return fail(FE_STATUS_INVALID, "at least one drafted token");
  if (drafts > kMaxDrafts)
    return fail(FE_STATUS_UNSUPPORTED, "at most %lld drafted tokens per call", (long long)kMaxDrafts);
  if (q_heads / c->kv_heads > kMaxGroup)
    return fail(FE_STATUS_UNSUPPORTED, "at most %lld query heads per KV head", (long long)kMaxGroup);
  return FE_STATUS_OK;
}

// Rows of [batch, heads, tokens, channels] can be read 16 bytes at a time.
bool rows_are_vectors(const void* p, const int64_t* s, int64_t batch, int64_t heads, int64_t tokens, int64_t channels) {
  return channels % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && (batch == 1 || s[0] % 8 == 0) &&
         (heads == 1 || s[1] % 8 == 0) && (tokens == 1 || s[2] % 8 == 0);
}

// Rows of [batch, drafts, drafts] mask bytes, the same.
int mask_is_vectors(const void* tree, int64_t batch_stride, int64_t drafts) {
  return tree && drafts % 16 == 0 && reinterpret_cast<uintptr_t>(tree) % 16 == 0 && batch_stride % 16 == 0;
}

int64_t round_up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// Geometry of a tree-attention launch: a function of the shapes alone, so the
// workspace query and the launch agree.
struct TreeGeometry {
  int heads, tile_rows, rows;  // query heads and rows per tile, rows per work item
  bool dual, cluster;
  int64_t M, MT, R, D4, ctas, slots, off_acc, bytes;
};

int tree_geometry(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t drafts, int64_t capacity,
                  int64_t channels, int sms, TreeGeometry* g) {
  const int64_t nbh = batch * kv_heads;
  const int64_t group = q_heads / kv_heads;
  g->M = group * drafts;
  g->heads = (int)std::min<int64_t>(group, 128 / drafts);
  g->tile_rows = g->heads * (int)drafts;
  g->dual = channels <= 128 && group > g->heads;
  g->rows = (g->dual ? 2 : 1) * g->tile_rows;
  g->MT = (g->M + g->rows - 1) / g->rows;
  g->R = std::min<int64_t>(g->M, g->rows);
  g->D4 = round_up(channels, 4);
  const int64_t tiles = (capacity + fe::DEC_TILE - 1) / fe::DEC_TILE + 1;
  if (nbh * g->MT * tiles > 0x3fffffff) return fail(FE_STATUS_UNSUPPORTED, "problem too large");
  g->ctas = std::min<int64_t>(sms, nbh * g->MT * tiles);
  // A cluster of eight per item instead of all SMs and a second launch: about
  // 4 us less, for (tiles/8 - items*tiles/SMs) more tiles of 1.2 us in a row.
  // (8 rows, one token: 4000 keys 12.1 us against 16.6, 6000 keys 13.9 and 15.2,
  // 8000 keys 16.5 and 17.1.)
  const int64_t items = nbh * g->MT;
  g->cluster = !g->dual && items * (fe::TREE_CLUSTER + 1) <= sms &&
               2 * tiles * (sms - items * fe::TREE_CLUSTER) <= 7 * fe::TREE_CLUSTER * sms;
  g->slots = nbh * g->MT + g->ctas;
  g->off_acc = round_up(g->slots * g->R * 8, 256);
  g->bytes = g->cluster ? 0 : g->off_acc + g->slots * g->R * g->D4 * 4;
  return FE_STATUS_OK;
}

// setmaxnreg draws on the registers a block was launched with (see launch_fwd).
template <typename Kern>
int check_regs(Kern kern, std::atomic<int>& checked, int needed, const char* what) {
  int regs = checked.load(std::memory_order_relaxed);
  if (regs == 0) {
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes");
    regs = fa.numRegs;
    checked.store(regs, std::memory_order_relaxed);
  }
  if (regs < needed)
    return fail(FE_STATUS_UNSUPPORTED, "%s kernel compiled with %d registers/thread, needs %d", what, regs, needed);
  return FE_STATUS_OK;
}

// Launches with programmatic stream serialization (the kernel waits for what is
// before it in the stream by itself), in clusters of `cluster` CTAs.
template <typename Kern, typename... Args>
int launch_dependent(Kern kern, dim3 grid, dim3 block, int smem, int cluster, cudaStream_t stream, const char* what,
                     Args... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) return cuda_fail(e, what);
  return FE_STATUS_OK;
}

// Clusters of `ctas` eviction CTAs (one to an SM) that are resident at once: one
// stays within a GPC, so larger ones leave SMs over (clusters of four use 136 of
// a B200's 148 SMs, of eight fewer still).
int64_t resident_rows(int dev, int ctas) {
  static std::atomic<int> counts[kMaxDevices][fe::SHRINK_MAX_CLUSTER + 1];  // 0: not asked yet
  if (ctas == 1 || dev < 0 || dev >= kMaxDevices) return sm_count(dev) / ctas;
  int n = counts[dev][ctas].load(std::memory_order_relaxed);
  if (n) return n;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(fe::SHRINK_THREADS);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, fe::fe_shrink_kernel<true>, &cfg) != cudaSuccess) {
    cudaGetLastError();  // (a guess is as right, if slower)
    n = sm_count(dev) / ctas;
  }
  n = std::max(n, 1);
  counts[dev][ctas].store(n, std::memory_order_relaxed);
  return n;
}

template <bool BF16, int DP, bool DUAL, bool CLUSTER>
int launch_tree(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tkn, const CUtensorMap& tvn,
                const fe::TreeParams& p, cudaStream_t stream) {
  using C = fe::TreeCfg<DP, DUAL>;
  auto kern = fe::fe_tree_kernel<BF16, DP, DUAL, CLUSTER>;
  int rc = set_smem(kern, C::SMEM);
  if (rc) return rc;
  static std::atomic<int> checked_regs{0};
  if ((rc = check_regs(kern, checked_regs, fe::FWD_REGS_NEEDED, "tree attention"))) return rc;
  const int64_t items = (int64_t)p.B * p.Hkv * p.MT;
  rc = launch_dependent(kern, dim3((unsigned)(CLUSTER ? items * fe::TREE_CLUSTER : p.nctas)), dim3(C::THREADS), C::SMEM,
                        CLUSTER ? fe::TREE_CLUSTER : 1, stream, "tree attention launch", tq, tk, tv, tkn, tvn, p);
  if (rc || CLUSTER) return rc;
  // Warps that share a row's partials: one per two partials (about ctas / items
  // of them), as long as the blocks are all resident at once (two an SM).
  const int64_t groups = (p.D4 / 4 + fe::TREE_JOIN_QUADS - 1) / fe::TREE_JOIN_QUADS, pairs = p.R * groups;
  auto blocks = [&](int splits) {
    const int64_t per_block = 32 * (fe::TREE_JOIN_WARPS / splits);
    return (pairs + per_block - 1) / per_block;
  };
  int splits = 1;
  while (splits < fe::TREE_JOIN_WARPS && splits * 2 * items < p.nctas && blocks(2 * splits) * items <= 2 * p.nctas) splits *= 2;
  return launch_dependent(fe::fe_tree_join_kernel<BF16>, dim3((unsigned)items, (unsigned)blocks(splits)),
                          dim3(fe::TREE_JOIN_THREADS), 0, 1, stream, "tree join launch", p, C::QTILES * p.tile_rows, splits);
}

template <bool BF16>
int launch_tree_dim(int dp, const TreeGeometry& g, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                    const CUtensorMap& tkn, const CUtensorMap& tvn, const fe::TreeParams& p, cudaStream_t s) {
  if (dp == 64)
    return g.dual      ? launch_tree<BF16, 64, true, false>(tq, tk, tv, tkn, tvn, p, s)
           : g.cluster ? launch_tree<BF16, 64, false, true>(tq, tk, tv, tkn, tvn, p, s)
                       : launch_tree<BF16, 64, false, false>(tq, tk, tv, tkn, tvn, p, s);
  if (dp == 128)
    return g.dual      ? launch_tree<BF16, 128, true, false>(tq, tk, tv, tkn, tvn, p, s)
           : g.cluster ? launch_tree<BF16, 128, false, true>(tq, tk, tv, tkn, tvn, p, s)
                       : launch_tree<BF16, 128, false, false>(tq, tk, tv, tkn, tvn, p, s);
  return g.cluster ? launch_tree<BF16, 256, false, true>(tq, tk, tv, tkn, tvn, p, s)
                   : launch_tree<BF16, 256, false, false>(tq, tk, tv, tkn, tvn, p, s);
}

}  // namespace

extern "C" {

int fe_cache_prepare(fe_cache* cache) {
  g_err[0] = 0;
  int rc = check_cache(cache);
  if (rc) return rc;
  cache->maps_of = 0;
  CUtensorMap tk, tv;
  if ((rc = cache_maps(cache, &tk, &tv))) return rc;
  memcpy(cache->map_k, &tk, sizeof(tk));
  memcpy(cache->map_v, &tv, sizeof(tv));
  cache->maps_of = layout_hash(cache);
  return FE_STATUS_OK;
}

int64_t fe_tree_workspace_bytes(const fe_cache* cache, int64_t q_heads, int64_t drafts) {
  g_err[0] = 0;
  if (check_cache(cache) || check_drafts(cache, q_heads, drafts)) return -1;
  int dev = 0;
  cudaGetDevice(&dev);
  TreeGeometry g;
  if (tree_geometry(cache->batch, q_heads, cache->kv_heads, drafts, cache->capacity, cache->channels, sm_count(dev), &g))
    return -1;
  return g.bytes;
}

int fe_tree_attention(const fe_cache* cache, const void* q, const int64_t* q_strides, const void* k_new,
                      const int64_t* k_new_strides, const void* v_new, const int64_t* v_new_strides,
                      const uint8_t* tree, int64_t tree_batch_stride, void* out, float* lse, void* workspace,
                      int64_t workspace_bytes, int64_t q_heads, int64_t drafts, float scale, void* stream) {
  g_err[0] = 0;
  int rc = check_cache(cache);
  if (rc) return rc;
  if ((rc = check_drafts(cache, q_heads, drafts))) return rc;
  if (!q || !k_new || !v_new || !out || !lse || !q_strides || !k_new_strides || !v_new_strides)
    return fail(FE_STATUS_INVALID, "null pointer");
  if (!std::isfinite(scale)) return fail(FE_STATUS_INVALID, "scale must be finite");
  if (q_strides[3] != 1) return fail(FE_STATUS_UNSUPPORTED, "q: channel stride must be 1");
  if (tree_batch_stride < 0) return fail(FE_STATUS_INVALID, "tree_batch_stride must be nonnegative");
  if (reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(FE_STATUS_UNSUPPORTED, "out must be 16-byte and workspace 256-byte aligned");
  int dev = 0;
  if ((rc = enter(cache->k, stream, &dev))) return rc;
  const int64_t B = cache->batch, H = cache->kv_heads, D = cache->channels;
  TreeGeometry g;
  if ((rc = tree_geometry(B, q_heads, H, drafts, cache->capacity, D, sm_count(dev), &g))) return rc;
  if (workspace_bytes < g.bytes || (g.bytes > 0 && !workspace))
    return fail(FE_STATUS_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)g.bytes);
  CUtensorMap tq, tk, tv, tkn, tvn;
  if ((rc = make_map(&tq, q, q_strides, B, q_heads, drafts, D, cache->dtype, "q", (int)drafts, g.heads))) return rc;
  if ((rc = cache_maps(cache, &tk, &tv))) return rc;
  if ((rc = make_map(&tkn, k_new, k_new_strides, B, H, drafts, D, cache->dtype, "k_new"))) return rc;
  if ((rc = make_map(&tvn, v_new, v_new_strides, B, H, drafts, D, cache->dtype, "v_new"))) return rc;
  fe::TreeParams p;
  p.q = static_cast<const uint16_t*>(q);
  p.q_sb = q_strides[0], p.q_sh = q_strides[1], p.q_st = q_strides[2];
  p.k_new = static_cast<const uint16_t*>(k_new);
  p.kn_sb = k_new_strides[0], p.kn_sh = k_new_strides[1], p.kn_st = k_new_strides[2];
  p.v_new = static_cast<const uint16_t*>(v_new);
  p.vn_sb = v_new_strides[0], p.vn_sh = v_new_strides[1], p.vn_st = v_new_strides[2];
  p.tree = tree;
  p.tree_sb = tree_batch_stride;
  p.lengths = cache->lengths;
  p.out = static_cast<uint16_t*>(out);
  p.lse = lse;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.stats = reinterpret_cast<float2*>(ws);
  p.acc = reinterpret_cast<float4*>(ws + g.off_acc);
  p.B = (int)B;
  p.Hq = (int)q_heads;
  p.Hkv = (int)H;
  p.G = (int)(q_heads / H);
  p.T = (int)drafts;
  p.D = (int)D;
  p.capacity = (int)cache->capacity;
  p.M = (int)g.M;
  p.tile_rows = g.tile_rows;
  p.MT = (int)g.MT;
  p.R = (int)g.R;
  p.D4 = (int)g.D4;
  p.nctas = (int)g.ctas;
  p.sc = (float)((double)scale * 1.4426950408889634);
  p.timeout_ns = (uint64_t)g_watchdog_ns;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int dp = padded_dim(D);
  return cache->dtype == FE_DTYPE_BF16 ? launch_tree_dim<true>(dp, g, tq, tk, tv, tkn, tvn, p, s)
                                       : launch_tree_dim<false>(dp, g, tq, tk, tv, tkn, tvn, p, s);
}

}  // extern "C"

namespace {

// The cache and the cache its updated bookkeeping goes to.
int check_bookkeeping(const fe_cache* c, const fe_cache* out) {
  int rc = check_cache(c);
  if (rc) return rc;
  if ((rc = check_cache(out))) return rc;
  if (c->k != out->k || c->v != out->v || c->batch != out->batch || c->kv_heads != out->kv_heads ||
      c->capacity != out->capacity || c->channels != out->channels || c->dtype != out->dtype)
    return fail(FE_STATUS_INVALID, "out must be the same cache's k and v with other bookkeeping");
  for (int i = 0; i < 4; ++i)
    if (c->k_strides[i] != out->k_strides[i] || c->v_strides[i] != out->v_strides[i])
      return fail(FE_STATUS_INVALID, "out must be the same cache's k and v with other bookkeeping");
  if (!c->mass || !c->positions || !out->mass || !out->positions) return fail(FE_STATUS_INVALID, "the cache has no mass and positions");
  if (!c->norms != !out->norms) return fail(FE_STATUS_INVALID, "norms must be given in both caches or in neither");
  // Every array of its own or every array shared: a kernel writes one while it reads the other.
  const bool shared = c->mass == out->mass;
  if ((c->positions == out->positions) != shared || (c->lengths == out->lengths) != shared ||
      (c->norms && (c->norms == out->norms) != shared))
    return fail(FE_STATUS_INVALID, "out must share all of the cache's bookkeeping or none of it");
  return FE_STATUS_OK;
}

// Drafts' weights between launches, and (in place) the new lengths.
int64_t commit_workspace(const fe_cache* c, bool in_place, int64_t q_heads, int64_t drafts, int64_t max_accepted,
                         int64_t* off_lengths) {
  const int64_t nbh = c->batch * c->kv_heads;
  const int64_t rows = c->channels <= 128 ? fe::CommitCfg<128>::ROWS : fe::CommitCfg<256>::ROWS;
  const bool launches = q_heads / c->kv_heads * max_accepted > rows;
  *off_lengths = launches ? round_up(nbh * drafts * 4, 256) : 0;
  return *off_lengths + (in_place ? nbh * 4 : 0);
}

template <bool BF16, int DP, int PARTS>
int launch_commit_parts(const CUtensorMap& tk, const CUtensorMap& tkn, fe::CommitParams p, cudaStream_t stream) {
  using C = fe::CommitCfg<DP>;
  auto kern = fe::fe_commit_mass_kernel<BF16, DP, PARTS>;
  int rc = set_smem(kern, C::SMEM);
  if (rc) return rc;
  static std::atomic<int> checked_regs{0};
  if ((rc = check_regs(kern, checked_regs, fe::COMMIT_REGS_NEEDED, "commit"))) return rc;
  // The accepted count is on the device; A is its most.
  for (int64_t row0 = 0; row0 == 0 || row0 < (int64_t)p.A * p.G; row0 += C::ROWS) {
    p.row0 = (int)row0;
    p.last = row0 + C::ROWS >= (int64_t)p.A * p.G;
    // A row begins with the gather of its queries: two key tiles' time, and one
    // more for every 64 of them (batch of 16, 4 rows: 31.5 us with none, 29.6 with
    // 2; 256 rows over 131k 100, 97, and 92 with 6).
    p.extra = 2 + (int)(std::min<int64_t>((int64_t)p.A * p.G - row0, C::ROWS) / 64);
    rc = launch_dependent(kern, dim3((unsigned)p.nctas), dim3(C::THREADS), C::SMEM, 1, stream, "commit launch", tk, tkn, p);
    if (rc) return rc;
  }
  return FE_STATUS_OK;
}

// As many parts to a score (see the kernel) as leave 128 columns for the queries;
// 256 channels always four.  Equally heavy fp16 keys of score 40 lean by 5.0e-5 with
// 256 channels in one sum, 1.8e-5 in two, under 7.2e-6 in four.  That costs their runs
// of more than 32 queries time (256 over 65536 tokens: one sum 115 us, two 137, four
// 227); up to 128 channels (1.8e-5 in one sum) longer runs keep one (256 queries over
// 131072 tokens: 92 us, two sums 138).
template <bool BF16, int DP>
int launch_commit(const CUtensorMap& tk, const CUtensorMap& tkn, const fe::CommitParams& p, cudaStream_t stream) {
  const int64_t rows = (int64_t)p.A * p.G;
  if constexpr (DP <= 128) {
    if (rows > 64) return launch_commit_parts<BF16, DP, 1>(tk, tkn, p, stream);
    if (rows > 32) return launch_commit_parts<BF16, DP, 2>(tk, tkn, p, stream);
  }
  return launch_commit_parts<BF16, DP, 4>(tk, tkn, p, stream);
}

}  // namespace

extern "C" {

int64_t fe_commit_workspace_bytes(const fe_cache* cache, const fe_cache* out, int64_t q_heads, int64_t drafts,
                                  int64_t max_accepted) {
  g_err[0] = 0;
  if (check_bookkeeping(cache, out) || check_drafts(cache, q_heads, drafts)) return -1;
  int64_t off;
  return commit_workspace(cache, cache->mass == out->mass, q_heads, drafts, max_accepted, &off);
}

int fe_commit_tokens(const fe_cache* cache, const fe_cache* out, const void* q, const int64_t* q_strides,
                     const void* k_new, const int64_t* k_new_strides, const void* v_new, const int64_t* v_new_strides,
                     const uint8_t* tree, int64_t tree_batch_stride, const float* lse, const int32_t* accepted,
                     int64_t max_accepted, const int32_t* new_positions, void* workspace, int64_t workspace_bytes,
                     int64_t q_heads, int64_t drafts, float scale, float recency_decay, void* stream) {
  g_err[0] = 0;
  int rc = check_bookkeeping(cache, out);
  if (rc) return rc;
  if ((rc = check_drafts(cache, q_heads, drafts))) return rc;
  if (max_accepted < 1 || max_accepted > fe::COMMIT_MAX_ACCEPTED)
    return fail(FE_STATUS_INVALID, "max_accepted must be in [1, %d]", fe::COMMIT_MAX_ACCEPTED);
  if (!q || !k_new || !v_new || !lse || !accepted || !new_positions || !q_strides || !k_new_strides ||
      !v_new_strides)
    return fail(FE_STATUS_INVALID, "null pointer");
  if (!std::isfinite(scale)) return fail(FE_STATUS_INVALID, "scale must be finite");
  if (!std::isfinite(recency_decay) || recency_decay < 0)
    return fail(FE_STATUS_INVALID, "recency_decay must be finite and nonnegative");
  if (q_strides[3] != 1 || v_new_strides[3] != 1) return fail(FE_STATUS_UNSUPPORTED, "q and v_new: channel stride must be 1");
  if (tree_batch_stride < 0) return fail(FE_STATUS_INVALID, "tree_batch_stride must be nonnegative");
  const int64_t B = cache->batch, H = cache->kv_heads, D = cache->channels;
  int64_t off_lengths;
  const int64_t need = commit_workspace(cache, cache->mass == out->mass, q_heads, drafts, max_accepted, &off_lengths);
  if (workspace_bytes < need || (need > 0 && !workspace)) return fail(FE_STATUS_INVALID, "workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 4) return fail(FE_STATUS_UNSUPPORTED, "workspace must be 4-byte aligned");
  if (cache->mass == out->mass && !cache->sync) return fail(FE_STATUS_INVALID, "the cache has no sync word");
  const int64_t units = B * H * ((cache->capacity + fe::DEC_TILE - 1) / fe::DEC_TILE + 1);
  if (units > 0x3fffffff) return fail(FE_STATUS_UNSUPPORTED, "problem too large");
  int dev = 0;
  if ((rc = enter(cache->k, stream, &dev))) return rc;
  CUtensorMap tk, tkn;
  if ((rc = cache_maps(cache, &tk, nullptr))) return rc;
  if ((rc = make_map(&tkn, k_new, k_new_strides, B, H, drafts, D, cache->dtype, "k_new"))) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  fe::CommitParams p;
  p.q = static_cast<const uint16_t*>(q);
  p.q_sb = q_strides[0], p.q_sh = q_strides[1], p.q_st = q_strides[2];
  p.lse = lse;
  p.accepted = accepted;
  p.tree = tree;
  p.tree_sb = tree_batch_stride;
  p.lengths = cache->lengths;
  p.mass_in = cache->mass;
  p.norms_in = cache->norms;
  p.pos_in = cache->positions;
  p.mass_out = out->mass;
  p.norms_out = out->norms;
  p.pos_out = out->positions;
  p.new_mass = reinterpret_cast<float*>(ws);
  p.copy = cache->mass != out->mass;
  p.new_lengths = p.copy ? out->lengths : reinterpret_cast<int32_t*>(ws + off_lengths);
  p.len_out = out->lengths;
  p.sync = cache->sync;
  p.k_new = static_cast<const uint16_t*>(k_new);
  p.kn_sb = k_new_strides[0], p.kn_sh = k_new_strides[1], p.kn_st = k_new_strides[2];
  p.v_new = static_cast<const uint16_t*>(v_new);
  p.vn_sb = v_new_strides[0], p.vn_sh = v_new_strides[1], p.vn_st = v_new_strides[2];
  p.k = static_cast<uint16_t*>(cache->k);
  p.k_sb = cache->k_strides[0], p.k_sh = cache->k_strides[1], p.k_st = cache->k_strides[2];
  p.v = static_cast<uint16_t*>(cache->v);
  p.v_sb = cache->v_strides[0], p.v_sh = cache->v_strides[1], p.v_st = cache->v_strides[2];
  p.new_positions = new_positions;
  p.rows_vec = rows_are_vectors(k_new, k_new_strides, B, H, drafts, D) && rows_are_vectors(v_new, v_new_strides, B, H, drafts, D) &&
               rows_are_vectors(cache->k, cache->k_strides, B, H, cache->capacity, D) &&
               rows_are_vectors(cache->v, cache->v_strides, B, H, cache->capacity, D);
  p.B = (int)B;
  p.Hq = (int)q_heads;
  p.Hkv = (int)H;
  p.G = (int)(q_heads / H);
  p.T = (int)drafts;
  p.A = (int)max_accepted;
  p.D = (int)D;
  p.capacity = (int)cache->capacity;
  p.nctas = (int)std::min<int64_t>(sm_count(dev), units);
  p.row0 = 0;
  p.sc = (float)((double)scale * 1.4426950408889634);
  p.decay_log2 = (double)recency_decay * 1.4426950408889634;
  p.q_vec = rows_are_vectors(q, q_strides, B, q_heads, drafts, D) ? 1 : 0;
  p.tree_vec = mask_is_vectors(tree, tree_batch_stride, drafts);
  p.timeout_ns = (uint64_t)g_watchdog_ns;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int dp = padded_dim(D);
  const bool bf16 = cache->dtype == FE_DTYPE_BF16;
  rc = bf16 ? (dp == 64 ? launch_commit<true, 64>(tk, tkn, p, s)
                        : dp == 128 ? launch_commit<true, 128>(tk, tkn, p, s) : launch_commit<true, 256>(tk, tkn, p, s))
            : (dp == 64 ? launch_commit<false, 64>(tk, tkn, p, s)
                        : dp == 128 ? launch_commit<false, 128>(tk, tkn, p, s) : launch_commit<false, 256>(tk, tkn, p, s));
  return rc;
}

int64_t fe_evict_workspace_bytes(const fe_cache* cache, int64_t budget) {
  g_err[0] = 0;
  if (check_cache(cache)) return -1;
  if (budget < 1) {
    fail(FE_STATUS_INVALID, "budget must be positive");
    return -1;
  }
  // Holes and movers of every row: no more than either side of the budget.
  const int64_t list = std::max<int64_t>(1, std::min(budget, cache->capacity - budget));
  return cache->batch * cache->kv_heads * (list * 8 + 4);
}

int fe_evict_tokens(const fe_cache* cache, const fe_cache* out, int64_t budget, int64_t recent, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  int rc = check_bookkeeping(cache, out);
  if (rc) return rc;
  if (budget < 1) return fail(FE_STATUS_INVALID, "budget must be positive");
  if (recent < 0 || recent > budget) return fail(FE_STATUS_INVALID, "recent must be an integer in [0, budget]");
  if (!workspace) return fail(FE_STATUS_INVALID, "null pointer");
  const int64_t rows = cache->batch * cache->kv_heads, cap = cache->capacity;
  const int64_t list = std::max<int64_t>(1, std::min(budget, cap - budget));
  if (workspace_bytes < rows * (list * 8 + 4)) return fail(FE_STATUS_INVALID, "workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 4) return fail(FE_STATUS_UNSUPPORTED, "workspace must be 4-byte aligned");
  for (const int64_t* s : {cache->k_strides, cache->v_strides}) {
    if (s[3] != 1) return fail(FE_STATUS_UNSUPPORTED, "cache: channel stride must be 1");
    for (int i = 0; i < 3; ++i)
      if (s[i] < 0 || s[i] % 8) return fail(FE_STATUS_UNSUPPORTED, "cache: strides must be multiples of 8");
  }
  if (reinterpret_cast<uintptr_t>(cache->k) % 16 || reinterpret_cast<uintptr_t>(cache->v) % 16)
    return fail(FE_STATUS_UNSUPPORTED, "cache: base pointers must be 16-byte aligned");
  int dev = 0;
  if ((rc = enter(cache->k, stream, &dev))) return rc;
  if (budget >= cap && cache->mass == out->mass) return FE_STATUS_OK;  // nothing can be over the budget
  fe::ShrinkParams p;
  p.k = static_cast<uint8_t*>(cache->k);
  p.k_sb = cache->k_strides[0] * 2, p.k_sh = cache->k_strides[1] * 2, p.k_st = cache->k_strides[2] * 2;
  p.v = static_cast<uint8_t*>(cache->v);
  p.v_sb = cache->v_strides[0] * 2, p.v_sh = cache->v_strides[1] * 2, p.v_st = cache->v_strides[2] * 2;
  p.mass_in = cache->mass;
  p.norms_in = cache->norms;
  p.pos_in = cache->positions;
  p.len_in = cache->lengths;
  p.mass_out = out->mass;
  p.norms_out = out->norms;
  p.pos_out = out->positions;
  p.len_out = out->lengths;
  p.holes = static_cast<int32_t*>(workspace);
  p.movers = p.holes + rows * list;
  p.list = list;
  p.counts = nullptr;
  p.rows = (int)rows;
  p.Hkv = (int)cache->kv_heads;
  p.capacity = (int)cap;
  p.budget = (int)std::min(budget, cap);
  p.recent = (int)std::min<int64_t>(recent, 0x7fffffff);
  p.row_bytes = (int)cache->channels * 2;
  p.copy = cache->mass != out->mass;
  // CTAs per row: as many as hold the row's keys, and, from 8192 slots on (below,
  // the cluster's barriers cost more: 12.0 us with one CTA, 14.3 with two for 32
  // rows of 5000), more while they still have 2048 slots each and all rows'
  // clusters are resident at once (48 rows of 12000: 19.3 us with two, 28.9 with four).
  auto held = [&](int ctas) {
    return round_up((cap + ctas * fe::SHRINK_WARPS - 1) / (ctas * fe::SHRINK_WARPS), 32) * fe::SHRINK_WARPS;
  };
  int cl = 1;
  while (cl < fe::SHRINK_MAX_CLUSTER && held(cl) > fe::SHRINK_SMEM_KEYS) cl *= 2;
  while (cl < fe::SHRINK_MAX_CLUSTER && cap >= 8192 && cap / (2 * cl) >= 2048 && rows <= resident_rows(dev, 2 * cl)) cl *= 2;
  // A second launch for the moves where it may spare the busiest SM 256 KB of
  // reads and writes: a row's own CTAs share its moves, the launch's all rows'.
  // (Rows of 46000 to a quarter, four rows 38.7 us in one launch, 25.6 in two, 24
  // rows 69 and 63; to a 32nd, 64 rows, where it spares less, 48 and 50.)
  const int64_t sms = sm_count(dev), resident = resident_rows(dev, cl), waves = (rows + resident - 1) / resident;
  const bool two = list * p.row_bytes * 4 * (waves * sms - rows * cl) >= (int64_t(256) << 10) * cl * sms;
  if (two) p.counts = p.movers + rows * list;
  const bool smem_keys = held(cl) <= fe::SHRINK_SMEM_KEYS;
  p.hold_positions = smem_keys && recent > 0 && 2 * held(cl) <= fe::SHRINK_SMEM_KEYS;
  auto kern = smem_keys ? fe::fe_shrink_kernel<true> : fe::fe_shrink_kernel<false>;
  const int smem = smem_keys ? (int)(held(cl) * (p.hold_positions ? 8 : 4)) : 0;
  if (smem > 16384 && (rc = set_smem(kern, fe::SHRINK_SMEM_KEYS * 4))) return rc;
  if (rows * cl > 0x7fffffff) return fail(FE_STATUS_UNSUPPORTED, "too many rows");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  rc = launch_dependent(kern, dim3((unsigned)(rows * cl)), dim3(fe::SHRINK_THREADS), smem, cl, s, "cache eviction launch", p);
  if (rc || !two) return rc;
  return launch_dependent(fe::fe_shrink_move_kernel, dim3(sm_count(dev)), dim3(fe::MOVE_THREADS), 0, 1, s, "cache move launch", p);
}

}  // extern "C"
