// Quantised paged key-value cache: handles, argument checks and the C ABI.
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <new>

#include "../../include/chonk_b200.h"
#include "ck_kv.h"
#include "ck_kv.cuh"
#include "ck_kv_attn.cuh"
#include "ck_kv_prompt.cuh"

// ---------------------------------------------------------------------------
// Launches

namespace {

template <typename... KArgs, typename... Args>
cudaError_t kv_launch_cluster(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, int cs, cudaStream_t s, bool pdl,
                              Args... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  int na = 0;
  if (pdl) {
    at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[na++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cs > 1) {
    at[na].id = cudaLaunchAttributeClusterDimension;
    at[na].val.clusterDim.x = cs;
    at[na].val.clusterDim.y = at[na].val.clusterDim.z = 1;
    na++;
  }
  cfg.attrs = at;
  cfg.numAttrs = na;
  return cudaLaunchKernelEx(&cfg, k, args...);
}
template <typename... KArgs, typename... Args>
cudaError_t kv_launch(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool pdl, Args... args) {
  return kv_launch_cluster(k, grid, block, smem, 1, s, pdl, args...);
}

}  // namespace

size_t kv_pool_bytes(const KvPool& p) {
  return (size_t)p.n_blocks * p.kvh * (p.block / KV_TILE) * kv_record_bytes(p.hd, p.vbits);
}


#define KV_STORE_WARPS 4096  // warps that a write spreads its tokens over, a token's rows among up to 8
#define KVP_SPLIT_TILES 8    // position tiles of a CTA, at least, where a prompt's cached positions are split
#define KV_UNIT_PAIRS 256    // pairs of records of a unit, at most, for one-token attention by unit
#define KV_CTA_PAIRS 64      // and of each of its CTAs

#define KV_EACH(X) X(64, 8) X(64, 4) X(128, 8) X(128, 4) X(256, 8) X(256, 4)

// warps of an SM in the form by list
static int kv_token_warps(int hd, int vb) {
#define KV_CASE(HD, VB) if (hd == HD && vb == VB) return KvTok<HD, VB>::WARPS;
  KV_EACH(KV_CASE)
#undef KV_CASE
  return 0;
}

// Workspace.  One token: two partial outputs of 8 heads per share (one per
// warp of the device), the prefix sums of a launch's queries and the partials'
// (m, l).  Prompts take no more: a split launch has at most one CTA per SM, of
// as many rows (16 x sms x 128 for 128 and 256 wide heads, twice that at 64 of
// which a CTA needs 256), a descriptor of 16 bytes a CTA in the place of the
// prefix sums.
void kv_workspace(const KvPool& p, int sms, size_t* part_bytes, size_t* ml_bytes) {
  const size_t slots = (size_t)sms * (p.hd == 256 ? 16 : 32);
  *part_bytes = slots * 8 * p.hd * sizeof(float);
  *ml_bytes = KV_PRE * sizeof(long long) + slots * 8 * sizeof(float2);
}

// the forms of k_kv_token
template <int HD, int VB, bool FINE>
struct KvForms {
  using C = KvTok<HD, VB>;
  static constexpr auto list = k_kv_token<HD, VB, false, C::WARPS, C::STAGES, FINE>;
  // by unit: 4 warps where the units fill the device, else 8 in up to 8 CTAs
  static constexpr int ST4 = HD == 256 ? 1 : 2, ST8 = HD == 256 ? 1 : 2;
  static constexpr auto unit4 = k_kv_token<HD, VB, true, 4, ST4, FINE>;
  static constexpr auto unit8 = k_kv_token<HD, VB, true, 8, ST8, FINE>;
  static constexpr int SUM = 8 * HD * 4;   // a CTA's sum
  static constexpr int SMEM4 = 4 * ST4 * C::PAIR_BYTES + SUM, SMEM8 = 8 * ST8 * C::PAIR_BYTES + SUM;
  static cudaError_t setup(KvDev* d) {
    cudaError_t e = cudaFuncSetAttribute(list, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(unit4, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM4);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(unit8, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM8);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(k_kv_prompt<HD, VB, FINE>, cudaFuncAttributeMaxDynamicSharedMemorySize, KvPr<HD, VB, FINE>::SMEM);
    return e == cudaSuccess ? fit(d) : e;
  }
  // clusters of unit8 that run at once: they lie within a GPC, so fewer than SMs / size
  static cudaError_t fit(KvDev* d) {
    for (int i = 0; i < 4; i++) {
      cudaLaunchConfig_t cfg;
      memset(&cfg, 0, sizeof cfg);
      cfg.gridDim = dim3(1 << i);
      cfg.blockDim = dim3(256);
      cfg.dynamicSmemBytes = SMEM8;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = 1 << i;
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      const cudaError_t e = cudaOccupancyMaxActiveClusters(&d->clusters[i], unit8, &cfg);
      if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
  }
  // pairs: most pairs of records that a unit can have (the block table's width
  // and the window stand for the lengths, which only the device knows).
  // *listed: whether the list was taken (its parts want joining).  By unit costs
  // one launch instead of two, by list balances.  Measured (us by unit, by
  // list), lengths from a third of the longest up: at head_dim 128 one query of
  // 2 units over up to 4000 positions 9.8 and 11.2; 16 of 2 units (4 CTAs each)
  // over 4000 12.4 and 17.8, over 8000 18.5 and 21.9; 64 of 8 units (a CTA each)
  // over 1040 29.3 and 29.6, over 2000 48.4 and 48.1, over 8000 153 and 134; at
  // head_dim 256 64 of one unit over 2000 17.6 and 28.0.  One bound serves all,
  // and at its end it is not every call's best: one query of 2 units over 8000
  // takes 12.8 and 11.8.  Clusters that do not all run at once make a second
  // wave: 16 of 8 CTAs, where 15 fit, took 12.4, in clusters of 4 8.0
  static cudaError_t launch(const KvAttn& a, int units, long long pairs, const KvDev& d, cudaStream_t s, bool pdl,
                            bool* listed) {
    const long long n = (long long)a.n * units;
    int lc = 0;   // log2 of a unit's CTAs: more while SMs are idle and a warp has more than one pair
    while (lc < 3 && (n << (lc + 1)) <= d.sms && n <= d.clusters[lc + 1] && (8 << lc) < pairs) lc++;
    const int cs = 1 << lc;
    *listed = pairs > KV_UNIT_PAIRS || pairs > KV_CTA_PAIRS * cs;
    if (*listed) return kv_launch(list, dim3(d.sms), dim3(C::WARPS * 32), C::SMEM, s, pdl, a, 1);
    if (n >= 2 * d.sms) return kv_launch(unit4, dim3((unsigned)n), dim3(128), SMEM4, s, pdl, a, 1);
    return kv_launch_cluster(unit8, dim3((unsigned)(n * cs)), dim3(256), SMEM8, cs, s, pdl, a, cs);
  }
};

cudaError_t kv_setup(const KvPool& p, int device, KvDev* d) {
  const cudaError_t e = cudaDeviceGetAttribute(&d->sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return e;
  // (both kinds of a form have the same bounds and shared memory: one answer for their clusters)
#define KV_CASE(HD, VB)                              \
  if (p.hd == HD && p.vbits == VB) {                 \
    const cudaError_t f = KvForms<HD, VB, true>::setup(d); \
    return f != cudaSuccess ? f : KvForms<HD, VB, false>::setup(d); \
  }
  KV_EACH(KV_CASE)
#undef KV_CASE
  return cudaErrorInvalidValue;
}

cudaError_t kv_store_launch(const KvStore& a, cudaStream_t s, bool pdl) {
  if (a.n == 0) return cudaSuccess;
  const int vec = (kv_vec8(a.q) ? 1 : 0) | (kv_vec8(a.k) ? 2 : 0) | (kv_vec8(a.v) ? 4 : 0) | (kv_vec8(a.qo) ? 8 : 0);
  // warps of a token: enough for a few warps on every scheduler, at most one a row
  const int rows = (a.heads + 2 * a.pool.kvh) * a.pool.hd / 512;
  int lw = 0;
  while (lw < 3 && (1 << lw) < rows && ((long long)a.n << lw) < KV_STORE_WARPS) lw++;
  const dim3 grid((unsigned)((((long long)a.n << lw) + 7) / 8)), block(KV_STORE_THREADS);
#define KV_CASE(HD, VB)                                                                                                 \
  if (a.pool.hd == HD && a.pool.vbits == VB)                                                                            \
    return a.k.type == KV_F32   ? kv_launch(k_kv_store<HD, VB, KV_F32>, grid, block, 0, s, pdl, a, vec, lw)            \
           : a.k.type == KV_F16 ? kv_launch(k_kv_store<HD, VB, KV_F16>, grid, block, 0, s, pdl, a, vec, lw)            \
                                : kv_launch(k_kv_store<HD, VB, KV_BF16>, grid, block, 0, s, pdl, a, vec, lw);
  KV_EACH(KV_CASE)
#undef KV_CASE
  return cudaErrorInvalidValue;
}

cudaError_t kv_load_launch(const KvLoad& a, cudaStream_t s) {
  if (a.n == 0) return cudaSuccess;
  const int vec = (kv_vec8(a.k) ? 1 : 0) | (kv_vec8(a.v) ? 2 : 0);
  const dim3 grid((a.n + KV_LOAD_THREADS / 32 - 1) / (KV_LOAD_THREADS / 32)), block(KV_LOAD_THREADS);
#define KV_CASE(HD, VB)                                                                                      \
  if (a.pool.hd == HD && a.pool.vbits == VB)                                                                 \
    return a.k.type == KV_F32   ? kv_launch(k_kv_load<HD, VB, KV_F32>, grid, block, 0, s, false, a, vec)     \
           : a.k.type == KV_F16 ? kv_launch(k_kv_load<HD, VB, KV_F16>, grid, block, 0, s, false, a, vec)     \
                                : kv_launch(k_kv_load<HD, VB, KV_BF16>, grid, block, 0, s, false, a, vec);
  KV_EACH(KV_CASE)
#undef KV_CASE
  return cudaErrorInvalidValue;
}

cudaError_t kv_attend_launch(const KvAttn& all, const KvDev& d, cudaStream_t s, bool pdl) {
  if (all.n_dev && all.n > KV_MAXQ) return cudaErrorInvalidValue;
  const int warps = d.sms * kv_token_warps(all.pool.hd, all.pool.vbits), units = kv_units(all.heads, all.pool.kvh);
  for (int i0 = 0; i0 < all.n; i0 += KV_MAXQ) {
    KvAttn a = all;
    a.n = all.n - i0 < KV_MAXQ ? all.n - i0 : KV_MAXQ;
    a.len += i0;
    if (a.seq) a.seq += i0;
    else if (i0) { a.tab.dev += (size_t)i0 * a.tab.max_blocks; a.tab.n_seqs -= i0; }
    a.q.p = (char*)a.q.p + (size_t)i0 * a.q.st * 2;
    a.o.p = (char*)a.o.p + (size_t)i0 * a.o.st * 2;
    // most pairs of records of a unit: the block table's width and the window bound them
    long long pairs = ((long long)a.tab.max_blocks * a.pool.block + KV_PAIR - 1) / KV_PAIR;
    if (a.window > 0 && pairs > a.window / KV_PAIR + 2) pairs = a.window / KV_PAIR + 2;
    bool listed = false;
    cudaError_t e = cudaErrorInvalidValue;
#define KV_CASE(HD, VB)                                                                                  \
  if (a.pool.hd == HD && a.pool.vbits == VB)                                                             \
    e = a.o.type == KV_F16 ? KvForms<HD, VB, true>::launch(a, units, pairs, d, s, pdl, &listed)          \
                           : KvForms<HD, VB, false>::launch(a, units, pairs, d, s, pdl, &listed);
    KV_EACH(KV_CASE)
#undef KV_CASE
    if (e != cudaSuccess) return e;
    if (!listed) continue;
    // a head's CTAs in the join (each some of its dims) while there are fewer
    // than SMs; thread groups: about half the partials that a unit has when all
    // are alike
    int z = 1;
    while (a.pool.hd / 4 / (2 * z) >= 8 && 2LL * z * a.n * a.heads <= d.sms) z *= 2;
    const int l = a.pool.hd / 4 / z, most = 1024 / l;
    int rows = l < 32 ? 32 / l : 1;
    while (rows < most && 2LL * rows * a.n * units < warps) rows *= 2;
    const dim3 grid(a.n, a.heads, z), block(rows * l);
    e = cudaErrorInvalidValue;
#define KV_JOIN(HD, L) if (a.pool.hd == HD && l == L) e = kv_launch(k_kv_join<HD, L>, grid, block, 0, s, true, a, warps);
    KV_JOIN(64, 16) KV_JOIN(64, 8) KV_JOIN(128, 32) KV_JOIN(128, 16) KV_JOIN(128, 8) KV_JOIN(256, 64) KV_JOIN(256, 32)
    KV_JOIN(256, 16) KV_JOIN(256, 8)
#undef KV_JOIN
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
cudaError_t kv_prompt_launch(const KvAttn& all, int sms, cudaStream_t s) {
  if (all.rows == 0) return cudaSuccess;
  const int gsz = all.heads / all.pool.kvh, hb = (gsz + 127) / 128, gs = (gsz + hb - 1) / hb;   // heads of a unit
  const int units = all.pool.kvh * hb, bt = (all.pool.hd == 256 ? 128 : 256) / gs, pt = 64;
  for (int i0 = 0; i0 < all.n; i0 += KVP_MAXS) {
    KvAttn a = all;
    a.n = all.n - i0 < KVP_MAXS ? all.n - i0 : KVP_MAXS;
    a.len += i0;
    a.cu += i0;
    a.tab.dev += (size_t)i0 * a.tab.max_blocks;
    a.tab.n_seqs -= i0;
    // tiles: at most a partial one per sequence.  The cached length is split
    // when they leave more than half of the SMs idle: what can be split (the
    // block table's width) into at least KVP_SPLIT_TILES position tiles a CTA
    const long long ctas = ((long long)a.rows / bt + a.n) * units;
    const long long tiles = ((long long)a.tab.max_blocks * a.pool.block + pt - 1) / pt;
    long long splits = ctas ? sms / ctas : 1;
    if (splits > tiles / KVP_SPLIT_TILES) splits = tiles / KVP_SPLIT_TILES;
    if (splits < 1) splits = 1;
    if (ctas * splits > 0x7fffffffLL) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)(ctas * splits));
    const int ends = (i0 == 0 ? 1 : 0) | (i0 + a.n == all.n ? 2 : 0);
    cudaError_t e = cudaErrorInvalidValue;
#define KV_PROMPT(HD, VB, FINE)                                                                                          \
  kv_launch(k_kv_prompt<HD, VB, FINE>, grid, dim3(KvPr<HD, VB, FINE>::THREADS), KvPr<HD, VB, FINE>::SMEM, s, false, a, \
            units, gs, (int)splits, ends)
#define KV_CASE(HD, VB)                      \
  if (a.pool.hd == HD && a.pool.vbits == VB) \
    e = a.o.type == KV_F16 ? KV_PROMPT(HD, VB, true) : KV_PROMPT(HD, VB, false);
    KV_EACH(KV_CASE)
#undef KV_PROMPT
#undef KV_CASE
    if (e != cudaSuccess) return e;
    if (splits > 1) {
      const dim3 jg((unsigned)ctas, bt * gs / 8 + (bt * gs % 8 != 0));
      if (a.pool.hd == 64) e = kv_launch(k_kv_prompt_join<64>, jg, dim3(256), 0, s, true, a, units, gs, (int)splits);
      else if (a.pool.hd == 128) e = kv_launch(k_kv_prompt_join<128>, jg, dim3(256), 0, s, true, a, units, gs, (int)splits);
      else e = kv_launch(k_kv_prompt_join<256>, jg, dim3(256), 0, s, true, a, units, gs, (int)splits);
      if (e != cudaSuccess) return e;
    }
  }
  return cudaSuccess;
}

// ---------------------------------------------------------------------------
// Handles

struct ck_kv {
  ck_kv_cfg cfg;
  int device;
  KvDev dev;
  KvPool pool;
  float *part, *ml;
  char err[256];

  int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(err, sizeof err, fmt, ap);
    va_end(ap);
    return code;
  }
};

namespace {

// The caller's current device is put back when a call ends.
struct OnDevice {
  int was = -1;
  cudaError_t rc;
  explicit OnDevice(int dev) {
    rc = cudaGetDevice(&was);
    if (rc == cudaSuccess && was != dev) rc = cudaSetDevice(dev);
    else if (rc == cudaSuccess) was = -1;
  }
  ~OnDevice() { if (was >= 0) cudaSetDevice(was); }
};

int kv_global(int code, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return ck_global_message(code, buf);
}

int type_bytes(int t) { return t == CK_DT_F32 ? 4 : 2; }

// token rows: present, of a known type, aligned to their elements
int check_rows(ck_kv* h, const char* call, const char* name, const ck_kv_rows& r, int n, bool f32, KvRows* out) {
  if (!r.dev && n > 0) return h->fail(CK_EINVAL, "%s: %s is null", call, name);
  if (r.dtype != CK_DT_F16 && r.dtype != CK_DT_BF16 && !(f32 && r.dtype == CK_DT_F32))
    return h->fail(CK_EINVAL, "%s: %s has type %d, expected %s", call, name, r.dtype, f32 ? "f32, f16 or bf16" : "f16 or bf16");
  if ((uintptr_t)r.dev % type_bytes(r.dtype)) return h->fail(CK_EINVAL, "%s: %s is not aligned to its elements", call, name);
  if (r.token_stride < 0 || r.head_stride < 0) return h->fail(CK_EINVAL, "%s: %s has a negative stride", call, name);
  out->p = r.dev;
  out->st = r.token_stride;
  out->sh = r.head_stride;
  out->type = r.dtype;
  return CK_OK;
}

// rows that are written: no two of them may overlap
int check_out(ck_kv* h, const char* call, const char* name, const ck_kv_rows& r, int n, int heads) {
  const int64_t hd = h->cfg.head_dim;
  const bool token_major = r.head_stride >= hd && (n < 2 || r.token_stride >= (heads - 1) * r.head_stride + hd);
  const bool head_major = r.token_stride >= hd && (heads < 2 || r.head_stride >= (n - 1) * r.token_stride + hd);
  if (n > 0 && !(heads == 1 && n == 1) && !token_major && !head_major)
    return h->fail(CK_EINVAL, "%s: rows of %s overlap (strides %lld, %lld)", call, name, (long long)r.token_stride,
                   (long long)r.head_stride);
  return CK_OK;
}

int check_table(ck_kv* h, const char* call, const ck_kv_table& t, KvTable* out) {
  if (t.n_seqs < 0 || t.max_blocks < 0 || (!t.dev && (int64_t)t.n_seqs * t.max_blocks > 0))
    return h->fail(CK_EINVAL, "%s: bad block table", call);
  if ((int64_t)t.max_blocks * h->cfg.block > INT32_MAX - KV_TILE)
    return h->fail(CK_EINVAL, "%s: %d blocks of %d positions pass the largest position", call, t.max_blocks, h->cfg.block);
  out->dev = t.dev;
  out->n_seqs = t.n_seqs;
  out->max_blocks = t.max_blocks;
  return CK_OK;
}

#define KVC(call)                                                                                            \
  do {                                                                                                       \
    cudaError_t e_ = (call);                                                                                 \
    if (e_ != cudaSuccess) return h->fail(CK_ECUDA, "%s: %s", #call, cudaGetErrorString(e_));                \
  } while (0)

}  // namespace

extern "C" {

int ck_kv_create(const ck_kv_cfg* cfg, int device, ck_kv** out) {
  if (!cfg || !out) return kv_global(CK_EINVAL, "ck_kv_create: bad argument");
  *out = nullptr;
  if (cfg->head_dim != 64 && cfg->head_dim != 128 && cfg->head_dim != 256)
    return kv_global(CK_EINVAL, "ck_kv_create: head_dim %d, expected 64, 128 or 256", cfg->head_dim);
  if (cfg->kv_heads < 1 || cfg->heads < cfg->kv_heads || cfg->heads > 1024 || cfg->heads % cfg->kv_heads)
    return kv_global(CK_EINVAL, "ck_kv_create: %d heads over %d kv heads", cfg->heads, cfg->kv_heads);
  if (cfg->block != 16 && cfg->block != 32 && cfg->block != 64 && cfg->block != 128)
    return kv_global(CK_EINVAL, "ck_kv_create: blocks of %d positions, expected 16, 32, 64 or 128", cfg->block);
  if (cfg->v_bits != 8 && cfg->v_bits != 4)
    return kv_global(CK_EINVAL, "ck_kv_create: values of %d bits, expected 8 or 4", cfg->v_bits);
  if (cfg->n_blocks < 1) return kv_global(CK_EINVAL, "ck_kv_create: %d blocks", cfg->n_blocks);
  ck_kv* h = new (std::nothrow) ck_kv();
  if (!h) return kv_global(CK_ENOMEM, "ck_kv_create: out of host memory");
  h->cfg = *cfg;
  h->device = device;
  KvPool& p = h->pool;
  p.n_blocks = cfg->n_blocks;
  p.kvh = cfg->kv_heads;
  p.block = cfg->block;
  p.hd = cfg->head_dim;
  p.vbits = cfg->v_bits;
  OnDevice on(device);
  auto bail = [&](int code, const char* what, cudaError_t e) {
    cudaGetLastError();
    cudaFree(p.base);
    cudaFree(p.err);
    cudaFree(h->part);
    cudaFree(h->ml);
    delete h;
    return kv_global(code, "ck_kv_create: %s: %s", what, cudaGetErrorString(e));
  };
  if (on.rc != cudaSuccess) return bail(CK_ECUDA, "device", on.rc);
  cudaError_t e = kv_setup(p, device, &h->dev);
  if (e != cudaSuccess) return bail(CK_ECUDA, "set-up", e);
  size_t pb = 0, mb = 0;
  kv_workspace(p, h->dev.sms, &pb, &mb);
  if ((e = cudaMalloc(&p.base, kv_pool_bytes(p))) != cudaSuccess || (e = cudaMalloc(&p.err, 16)) != cudaSuccess ||
      (e = cudaMalloc(&h->part, pb)) != cudaSuccess || (e = cudaMalloc(&h->ml, mb)) != cudaSuccess)
    return bail(CK_ENOMEM, "cudaMalloc", e);
  if ((e = cudaMemset(p.err, 0, 16)) != cudaSuccess || (e = cudaDeviceSynchronize()) != cudaSuccess)
    return bail(CK_ECUDA, "set-up", e);
  *out = h;
  return CK_OK;
}

int ck_kv_destroy(ck_kv* h) {
  if (!h) return CK_OK;
  OnDevice on(h->device);
  cudaFree(h->pool.base);   // waits for the device's work
  cudaFree(h->pool.err);
  cudaFree(h->part);
  cudaFree(h->ml);
  delete h;
  return CK_OK;
}

const char* ck_kv_last_error(ck_kv* h) { return h ? h->err : ck_global_error(); }

int ck_kv_bytes(ck_kv* h, size_t* pool_bytes) {
  if (!h || !pool_bytes) return kv_global(CK_EINVAL, "ck_kv_bytes: bad argument");
  *pool_bytes = kv_pool_bytes(h->pool);
  return CK_OK;
}

int ck_kv_store(ck_kv* h, const ck_kv_store_args* a, void* stream) {
  if (!h || !a) return kv_global(CK_EINVAL, "ck_kv_store: bad argument");
  if (a->n < 0 || (a->n > 0 && (!a->seq || !a->pos))) return h->fail(CK_EINVAL, "ck_kv_store: bad token list");
  KvStore p;
  memset(&p, 0, sizeof p);
  const int H = h->cfg.heads;
  int rc;
  if ((rc = check_rows(h, "ck_kv_store", "k", a->k, a->n, true, &p.k)) ||
      (rc = check_rows(h, "ck_kv_store", "v", a->v, a->n, true, &p.v)) ||
      (rc = check_table(h, "ck_kv_store", a->table, &p.tab)))
    return rc;
  if (a->q.dev) {
    if ((rc = check_rows(h, "ck_kv_store", "q", a->q, a->n, true, &p.q)) ||
        (rc = check_rows(h, "ck_kv_store", "q_out", a->q_out, a->n, false, &p.qo)) ||
        (rc = check_out(h, "ck_kv_store", "q_out", a->q_out, a->n, H)))
      return rc;
    p.heads = H;
  } else if (a->q_out.dev) {
    return h->fail(CK_EINVAL, "ck_kv_store: q_out without q");
  }
  if (a->k.dtype != a->v.dtype || (a->q.dev && a->q.dtype != a->k.dtype))
    return h->fail(CK_EINVAL, "ck_kv_store: q, k and v have to be of one type");
  if (!(a->eps >= 0.f && a->eps < INFINITY) && (a->q_norm || a->k_norm)) return h->fail(CK_EINVAL, "ck_kv_store: eps %g", a->eps);
  p.pool = h->pool;
  p.seq = a->seq;
  p.pos = a->pos;
  p.n = a->n;
  p.qw = a->q_norm;
  p.kw = a->k_norm;
  p.inv_freq = a->inv_freq;
  p.eps = a->eps;
  p.interleaved = a->interleaved ? 1 : 0;
  OnDevice on(h->device);
  KVC(on.rc);
  KVC(kv_store_launch(p, (cudaStream_t)stream, false));
  return CK_OK;
}

int ck_kv_load(ck_kv* h, const ck_kv_load_args* a, void* stream) {
  if (!h || !a) return kv_global(CK_EINVAL, "ck_kv_load: bad argument");
  if (a->n < 0 || (a->n > 0 && (!a->seq || !a->pos))) return h->fail(CK_EINVAL, "ck_kv_load: bad token list");
  KvLoad p;
  memset(&p, 0, sizeof p);
  const int K = h->cfg.kv_heads;
  int rc;
  if ((rc = check_rows(h, "ck_kv_load", "k", a->k, a->n, true, &p.k)) ||
      (rc = check_rows(h, "ck_kv_load", "v", a->v, a->n, true, &p.v)) ||
      (rc = check_out(h, "ck_kv_load", "k", a->k, a->n, K)) || (rc = check_out(h, "ck_kv_load", "v", a->v, a->n, K)) ||
      (rc = check_table(h, "ck_kv_load", a->table, &p.tab)))
    return rc;
  if (a->k.dtype != a->v.dtype) return h->fail(CK_EINVAL, "ck_kv_load: k and v have to be of one type");
  p.pool = h->pool;
  p.seq = a->seq;
  p.pos = a->pos;
  p.n = a->n;
  OnDevice on(h->device);
  KVC(on.rc);
  KVC(kv_load_launch(p, (cudaStream_t)stream));
  return CK_OK;
}

static int attn_args(ck_kv* h, const char* call, const ck_kv_attend_args* a, int rows, KvAttn* p) {
  memset(p, 0, sizeof *p);
  if (a->n < 0 || rows < 0 || (a->n > 0 && !a->len)) return h->fail(CK_EINVAL, "%s: bad length list", call);
  if (a->window < 0) return h->fail(CK_EINVAL, "%s: window %d", call, a->window);
  if (!(a->scale > -INFINITY && a->scale < INFINITY)) return h->fail(CK_EINVAL, "%s: scale is not finite", call);
  int rc;
  if ((rc = check_rows(h, call, "q", a->q, rows, false, &p->q)) ||
      (rc = check_rows(h, call, "out", a->out, rows, false, &p->o)) ||
      (rc = check_out(h, call, "out", a->out, rows, h->cfg.heads)) || (rc = check_table(h, call, a->table, &p->tab)))
    return rc;
  p->pool = h->pool;
  p->seq = a->seq;
  p->len = a->len;
  p->n = a->n;
  p->rows = rows;
  p->heads = h->cfg.heads;
  p->window = a->window;
  p->scale = a->scale;
  p->part = h->part;
  p->ml = h->ml;
  return CK_OK;
}

int ck_kv_attend(ck_kv* h, const ck_kv_attend_args* a, void* stream) {
  if (!h || !a) return kv_global(CK_EINVAL, "ck_kv_attend: bad argument");
  KvAttn p;
  int rc = attn_args(h, "ck_kv_attend", a, a->n, &p);
  if (rc) return rc;
  if (!a->seq && a->n > a->table.n_seqs)
    return h->fail(CK_EINVAL, "ck_kv_attend: %d queries for %d rows of the block table", a->n, a->table.n_seqs);
  OnDevice on(h->device);
  KVC(on.rc);
  KVC(kv_attend_launch(p, h->dev, (cudaStream_t)stream, false));
  return CK_OK;
}

int ck_kv_attend_prompt(ck_kv* h, const ck_kv_attend_args* a, const int32_t* cu, int rows, void* stream) {
  if (!h || !a) return kv_global(CK_EINVAL, "ck_kv_attend_prompt: bad argument");
  KvAttn p;
  int rc = attn_args(h, "ck_kv_attend_prompt", a, rows, &p);
  if (rc) return rc;
  if (a->seq) return h->fail(CK_EINVAL, "ck_kv_attend_prompt: sequence i reads row i of the block table");
  if (a->n > a->table.n_seqs)
    return h->fail(CK_EINVAL, "ck_kv_attend_prompt: %d sequences for %d rows of the block table", a->n, a->table.n_seqs);
  if (rows > 0 && (!cu || a->n < 1)) return h->fail(CK_EINVAL, "ck_kv_attend_prompt: bad row list");
  p.cu = cu;
  OnDevice on(h->device);
  KVC(on.rc);
  KVC(kv_prompt_launch(p, h->dev.sms, (cudaStream_t)stream));
  return CK_OK;
}

int ck_kv_check(ck_kv* h, void* stream) {
  if (!h) return kv_global(CK_EINVAL, "ck_kv_check: null cache");
  OnDevice on(h->device);
  KVC(on.rc);
  int bits = 0;
  cudaStream_t s = (cudaStream_t)stream;
  KVC(cudaMemcpyAsync(&bits, h->pool.err, sizeof bits, cudaMemcpyDeviceToHost, s));
  KVC(cudaStreamSynchronize(s));
  if (!bits) return CK_OK;
  KVC(cudaMemsetAsync(h->pool.err, 0, sizeof bits, s));
  KVC(cudaStreamSynchronize(s));
  return h->fail(CK_EDEVICE, "%s%s%s%s%s", bits & KV_ERR_SEQ ? "sequence outside the block table; " : "",
                 bits & KV_ERR_POS ? "position or length outside the block table; " : "",
                 bits & KV_ERR_BLOCK ? "block table entry outside the pool; " : "",
                 bits & KV_ERR_ROWS ? "prompt's sequence outside the query rows; " : "",
                 bits & KV_ERR_WAIT ? "device wait timed out; " : "");
}

}  // extern "C"
