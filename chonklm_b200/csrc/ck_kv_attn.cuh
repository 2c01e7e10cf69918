// Attention of one new token per sequence over the quantised paged cache.
//
//   s_j = scale * sum_g dk[j][g] * (q_g . ck[j][g])      (codes c, scales d per group g of 32)
//   o   = sum_j exp(s_j - m) * dv[j][g] * cv[j][g] / sum_j exp(s_j - m)
//
// Bound by the cache's bytes (and, close behind, by the instructions that turn
// codes into operands).  A unit is one query's up to 8 heads of one kv head;
// they share every record that is read.  A warp takes pairs of 16-position
// records, keeps several pairs in flight in its own part of shared memory (one
// cp.async.bulk per record, completing on the warp's mbarriers) and waits for
// no other warp.  Two ways to hand out the pairs:
//   by list   all units' visible pairs form one list, cut into equal shares,
//             one per warp of the device: ragged lengths balance by
//             themselves, one long sequence spreads over every SM, and no
//             length is needed on the host.  A unit that lies in one share is
//             finished by its warp; the others leave unnormalised partial
//             outputs with their (m, l), which k_kv_join adds in the order of
//             the shares (no atomics: the result does not depend on timing).
//   by unit   short caches: one CTA or one cluster of CTAs per unit, the
//             warps' parts added through shared memory, the CTAs' through
//             distributed shared memory; one launch.
// Measured at head_dim 128, 4-bit values: 64 sequences of 493 MB in all take
// 92 us by list (5.4 TB/s, 82 % of the copy bandwidth; 380 warp instructions
// a record, issue slots 62 % busy) and the join 8 more.  A warp a record, a
// row of heads as the product's rows, took 139 us: pairs halve the fixed work
// of a step, and the heads as columns waste none of the product's rows.  16 or
// 8 warps an SM instead of 12 took 105 and 119 us.
//
// Products run on m16n8k16 tensor instructions (a unit has 8 rows, too few for
// tcgen05's 64-row tiles), the heads as the 8 columns: S^T = K Q^T with 16
// positions as rows, O^T = V^T P^T with 16 dims as rows (P^T from S^T's
// accumulators by one 8x8 transposition in registers).  A key's byte c + 128
// is taken as the fp16 number (c + 128) 2^-24 (its bits as they are),
// -128 2^-24 sum(q) is where the sum begins, and each group's sum is
// multiplied by its scale in 32 bits.  A value's byte becomes fp16 by
// 0x6400 | byte = 1024 + byte.  Rounded to 16 bits: p = exp(s - m) (11 bits; l
// sums the rounded p, so that weights still add up to one) and, for bf16
// outputs, a value code * scale (11 of 18 bits, as an fp16 cache would hold it).
// FINE, for fp16 outputs, whose own rounding is small enough for that to show:
// the scale's upper bits and the rest are products of their own (KV_TOP; 4-bit
// values are exact then).  Over the fp16 cases the output is off by 1.01 to 1.08
// times what the same in 32 bits is, with one product by 1.1 to 1.8 times; 256
// short sequences at head_dim 64 take 13.7 us, 12.6 with one.
#pragma once
#include "ck_kv.cuh"

// prefix sums of a launch's queries sit in shared memory, and in the workspace
#define KV_PRE (KV_MAXQ + 2) // (keeps what follows 16-byte aligned)
#define KV_PAIR 32           // positions of a pair of records
#define KV_SLACK 6.f         // log2 that a score may exceed the reference maximum before o is rescaled
#define KV_BOOST 8.f         // p is kept times 2^8 (cancelled by l), so that small p stay normal fp16 numbers

// by list: one CTA per SM; the warps that the registers allow (accumulators:
// head_dim / 4 a thread) and the pairs that fit 209 KB
template <int HD, int VB>
struct KvTok {
  static constexpr int WARPS = HD == 256 ? (VB == 8 ? 6 : 8) : HD == 128 ? 12 : 16;
  static constexpr int PAIR_BYTES = 2 * KvRec<HD, VB>::BYTES;
  static constexpr int FIT = 209 * 1024 / WARPS / PAIR_BYTES, STAGES = FIT > 4 ? 4 : FIT;
  static constexpr int SMEM = WARPS * STAGES * PAIR_BYTES;
};

// d = a b + c
__device__ __forceinline__ void kv_mma_from(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// transposes an 8x8 matrix of 16-bit elements, two of a row in each thread
__device__ __forceinline__ uint32_t kv_transpose(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void kv_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// bytes (sel) of w as two fp16 numbers minus 1024 + bias
template <uint32_t SEL, int BIAS>
__device__ __forceinline__ uint32_t kv_half2(uint32_t w) {
  const uint32_t u = __byte_perm(w, 0x64646464u, SEL);
  const __half2 h = __hsub2(*(const __half2*)&u, __half2half2(__ushort_as_half((unsigned short)(0x6400 + BIAS))));
  return *(const uint32_t*)&h;
}
// codes of an fp16 pair 1024 + byte: byte - 128, or nibble - 8 of 4 bits (the
// low ones, or the high ones as (1024 + 16 x) / 16 - 72)
template <int VB>
__device__ __forceinline__ uint32_t kv_code2(uint32_t h, int nib) {
  __half2 v;
  if (VB == 8) {
    v = __hsub2(*(const __half2*)&h, __half2half2(__ushort_as_half(0x6480)));
  } else if (nib == 0) {
    const uint32_t x = h & 0xff0fff0fu;
    v = __hsub2(*(const __half2*)&x, __half2half2(__ushort_as_half(0x6408)));
  } else {
    const uint32_t x = h & 0xfff0fff0u;
    v = __hfma2(*(const __half2*)&x, __half2half2(__ushort_as_half(0x2c00)), __half2half2(__ushort_as_half(0xd480)));
  }
  return *(const uint32_t*)&v;
}
__device__ __forceinline__ uint32_t kv_hmul2(uint32_t a, uint32_t b) {
  const __half2 h = __hmul2(*(const __half2*)&a, *(const __half2*)&b);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t kv_pack2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// fp16 scales, all groups: of one position (W = HD / 64 words) or of two
// neighbouring ones
template <int W>
__device__ __forceinline__ void kv_lds(const uint8_t* p, uint32_t (&u)[W]) {
  if (W == 1) {
    u[0] = *(const uint32_t*)p;
  } else if (W == 2) {
    const uint2 x = *(const uint2*)p;
    u[0] = x.x; u[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; i++) {
      const uint4 x = *(const uint4*)(p + 16 * i);
      u[4 * i] = x.x; u[4 * i + 1] = x.y; u[4 * i + 2] = x.z; u[4 * i + 3] = x.w;
    }
  }
}
// the pair (group g of the first position, group g of the second)
template <int G, int W>
__device__ __forceinline__ uint32_t kv_scale_pair(const uint32_t (&u)[W], int g) {
  return __byte_perm(u[g >> 1], u[G / 2 + (g >> 1)], (g & 1) ? 0x7632 : 0x5410);
}

// visible pairs of records of a query: the first one and their number
__device__ __forceinline__ int kv_pairs(int len, int window, int& t0) {
  const int lo = window > 0 && len > window ? len - window : 0;
  t0 = lo / KV_PAIR;
  return len > 0 ? (len + KV_PAIR - 1) / KV_PAIR - t0 : 0;
}
__device__ __forceinline__ int kv_len(const KvAttn& A, int i) {
  const int len = A.len[i] + A.len_add;
  if (len > A.tab.max_blocks * A.pool.block) {
    atomicOr(A.pool.err, KV_ERR_POS);
    return 0;
  }
  if (len > 0 && A.seq && (unsigned)A.seq[i] >= (unsigned)A.tab.n_seqs) {
    atomicOr(A.pool.err, KV_ERR_SEQ);
    return 0;
  }
  return len > 0 ? len : 0;
}

// units per query (8 heads at most each) and shares' length
__host__ __device__ __forceinline__ int kv_units(int heads, int kvh) { return kvh * ((heads / kvh + 7) / 8); }
__device__ __forceinline__ long long kv_share(long long total, int warps) { return (total + warps - 1) / warps; }

// The partial outputs of a unit whose records are [a, a + tiles) of the list:
// a unit is the first one of every share it reaches into but its own first,
// where it is that only if it begins the share.
struct KvSlots {
  int s0, cnt;
  bool mid;
  __device__ __forceinline__ KvSlots(long long a, long long tiles, long long per) {
    const long long last = a + tiles - 1;
    if (last >> 32) {
      s0 = (int)(a / per);
      cnt = (int)(last / per) - s0 + 1;
    } else {                                   // (a 64-bit division is some 100 instructions)
      s0 = (int)((uint32_t)a / (uint32_t)per);
      cnt = (int)((uint32_t)last / (uint32_t)per) - s0 + 1;
    }
    mid = a > s0 * per;
  }
  __device__ __forceinline__ int slot(int k) const { return 2 * (s0 + k) + (k == 0 && mid ? 1 : 0); }
};

__device__ __forceinline__ uint32_t kv_cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void kv_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the same shared-memory address in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t kv_mapa(const void* p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float4 kv_ld_cluster4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float2 kv_ld_cluster2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// UNIT: by unit, W warps a CTA, ST stages each, `cs` CTAs a unit; else by list.
// FINE: values in two products.
template <int HD, int VB, bool UNIT, int W, int ST, bool FINE>
__global__ void __launch_bounds__(W * 32, UNIT ? (HD == 256 ? 8 : HD == 64 ? 24 : 16) / W : 1) k_kv_token(const __grid_constant__ KvAttn A, int cs) {
  using R = KvRec<HD, VB>;
  constexpr int G = R::G, NT = W * 32, EPT = (KV_MAXQ + NT - 1) / NT, PB = 2 * R::BYTES;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ long long pre[UNIT ? 1 : KV_MAXQ + 1];
  __shared__ long long wsum[W];
  __shared__ float2 uml[UNIT ? W : 1][8], cml[8];
  __shared__ __align__(8) uint64_t bars[W * ST];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gsz = A.heads / A.pool.kvh, HB = (gsz + 7) / 8, U = A.pool.kvh * HB;
  if (lane == 0)
    for (int i = 0; i < ST; i++) mbar_init(&bars[warp * ST + i], 1);
  mbar_fence_init();
  __syncwarp();
  pdl_wait();
  pdl_launch();
  const int n = A.n_dev ? min(*A.n_dev, A.n) : A.n;
  const int share = warp * gridDim.x + blockIdx.x;   // neighbouring shares go to different SMs
  float2* ml = (float2*)((long long*)A.ml + KV_PRE);
  // where a pair lies: query, unit of the query, pair of the sequence, the
  // unit's first pair and last + 1
  struct Place { int q, u, pair, beg, end; };
  Place f, c;                                // the pair to fetch next, and to compute next
  long long w0 = 0;
  int todo;                                  // pairs of this warp
  if (UNIT) {
    const int rank = blockIdx.x % cs, w = rank * W + warp, ws = cs * W;
    f.q = blockIdx.x / cs / U;
    f.u = blockIdx.x / cs % U;
    if (f.q >= n) return;
    const long long pairs = kv_pairs(kv_len(A, f.q), A.window, f.beg);
    f.end = f.beg + (int)pairs;
    f.pair = f.beg + (int)(pairs * w / ws);
    todo = f.beg + (int)(pairs * (w + 1) / ws) - f.pair;
  } else {
    // prefix sums of the queries' pairs over all their units
    long long mine[EPT], run = 0;
#pragma unroll
    for (int e = 0; e < EPT; e++) {
      const int i = tid * EPT + e;
      int t0;
      mine[e] = run;
      if (i < n) run += (long long)kv_pairs(kv_len(A, i), A.window, t0) * U;
    }
    long long inc = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    long long base = 0;
    for (int w = 0; w < warp; w++) base += wsum[w];
#pragma unroll
    for (int e = 0; e < EPT; e++)
      if (tid * EPT + e < KV_MAXQ) pre[tid * EPT + e] = base + inc - run + mine[e];
    if (tid == NT - 1) pre[KV_MAXQ] = base + inc;
    __syncthreads();
    if (blockIdx.x == 0)                     // for k_kv_join: prefix sums, then the (m, l) pairs
      for (int i = tid; i <= n; i += NT) ((long long*)A.ml)[i] = pre[i];
    const long long total = pre[KV_MAXQ], per = kv_share(total, gridDim.x * W);
    w0 = share * per;
    todo = (int)min(total - w0, per);
    if (todo <= 0) return;
  }
  auto locate = [&](int at, Place& p) {      // pair `at` of the share
    const long long x = w0 + at;
    int lo = 0, hi = n;                      // last query with pre[q] <= x (queries without pairs repeat a value)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= x) lo = mid; else hi = mid;
    }
    p.q = lo;
    const int pairs = kv_pairs(kv_len(A, lo), A.window, p.beg);
    const long long off = x - pre[lo];
    p.u = (int)(off / pairs);
    p.pair = p.beg + (int)(off % pairs);
    p.end = p.beg + pairs;
  };
  if (!UNIT) locate(0, f);
  c = f;

  uint8_t* st = ring + warp * ST * PB;
  uint64_t* bar = &bars[warp * ST];
  const int r = lane >> 2, t = lane & 3;
  const int lb = 31 - __clz(A.pool.block / KV_TILE), bmask = (1 << lb) - 1;   // records of a block: a power of two
  const size_t bstride = (size_t)A.pool.kvh * R::BYTES << lb;
  int fetched = 0, fstage = 0;
  int ids = 0, ids_at = -64;                 // block ids of the pairs ids_at .. ids_at + 15, two lanes a pair
  uint32_t bad = 0;                          // records that do not exist: bits 2 stage and 2 stage + 1
  auto issue = [&]() {
    if (fetched >= todo) return;
    if ((unsigned)(f.pair - ids_at) >= 16u) {
      ids_at = f.pair;
      const int seq = A.seq ? A.seq[f.q] : f.q, rec = 2 * f.pair + lane;
      ids = rec < A.tab.max_blocks << lb ? A.tab.dev[(size_t)seq * A.tab.max_blocks + (rec >> lb)] : -1;
      // the second record of the last pair may lie past the end, the first of the first one before the window (and its
      // block be another's by now): not read, masked like any place that is not seen
      const int len = kv_len(A, f.q);
      if (rec * KV_TILE >= len || (A.window > 0 && (rec + 1) * KV_TILE <= len - A.window)) ids = -2;
    }
    // lane 0 copies the first record, lane 1 the second
    const int id = __shfl_sync(0xffffffffu, ids, 2 * (f.pair - ids_at) + (lane & 1));
    const bool ok = lane < 2 && (unsigned)id < (unsigned)A.pool.n_blocks;
    const uint32_t have = __ballot_sync(0xffffffffu, ok);
    if (lane == 0) {
      if (have) mbar_expect_tx(bar + fstage, __popc(have) * R::BYTES);
      else mbar_arrive(bar + fstage);
    }
    __syncwarp();
    if (ok) {
      const int rec = 2 * f.pair + lane;
      bulk_g2s(st + fstage * PB + lane * R::BYTES,
               A.pool.base + ((size_t)(f.u / HB) * R::BYTES << lb) + id * bstride + (rec & bmask) * R::BYTES, R::BYTES,
               bar + fstage);
    } else if (lane < 2 && id != -2) {
      atomicOr(A.pool.err, KV_ERR_BLOCK);
    }
    bad = (bad & ~(3u << (2 * fstage))) | ((~have & 3u) << (2 * fstage));
    fstage = fstage + 1 == ST ? 0 : fstage + 1;
    fetched++;
    if (!UNIT && ++f.pair == f.end) {
      f.pair = f.beg;
      ids_at = -64;
      if (++f.u == U && fetched < todo) locate(fetched, f);
    } else if (UNIT) {
      f.pair++;
    }
  };
#pragma unroll
  for (int i = 0; i < ST; i++) issue();

  const bool vecq = (uintptr_t)A.q.p % 16 == 0 && A.q.st % 8 == 0 && A.q.sh % 8 == 0;
  const bool vec = kv_vec4(A.o);
  int cstage = 0, at = 0;
  uint32_t parity = 0;
  bool gave_up = false;
  while (UNIT || at < todo) {
    // one unit, or the part of it in this share
    const bool from_start = c.pair == c.beg;
    const int stop = min(todo, at + c.end - c.pair);
    const int len = kv_len(A, c.q), vis0 = A.window > 0 && len > A.window ? len - A.window : 0;
    const int kvh = c.u / HB, h0 = kvh * gsz + (c.u % HB) * 8, nh = min(8, gsz - (c.u % HB) * 8);
    // Q^T: columns = heads, the k index in the order of the codes' bytes:
    // thread t holds dims 8t .. 8t + 7 of each group of head r, two steps of 16
    uint32_t qa[G][4];
    float q0[G][4], sc[2];                   // heads 2t and 2t + 1: where each group's sum begins; scale to log2
    {
      const unsigned short* qp = (const unsigned short*)A.q.p + (size_t)c.q * A.q.st + (size_t)(h0 + r) * A.q.sh + 8 * t;
      float top = 0.f;
#pragma unroll
      for (int g = 0; g < G; g++) {
        uint32_t* x = qa[g];
        x[0] = x[1] = x[2] = x[3] = 0u;
        if (r < nh) {
          if (vecq) {
            const uint4 v = *(const uint4*)(qp + 32 * g);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = qp[32 * g + 2 * e] | ((uint32_t)qp[32 * g + 2 * e + 1] << 16);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 y = kv_pair16(x[e], A.q.type);
          top = fmaxf(top, fmaxf(fabsf(y.x), fabsf(y.y)));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // a power of two brings the row's largest value to [2^8, 2^9): fp16 then
      // holds a 16-bit q of either type to within 2^-33 of that value
      int e = (int)(__float_as_uint(top) >> 23) - 127;
      e = e > 127 ? 8 : max(e, -100);
      const float up = __uint_as_float((uint32_t)(127 + 8 - e) << 23);
      // 2^24: the codes' fp16 numbers.  Above 2^100 the factor is cut: no sum
      // that it multiplies passes 2^16, so that scores stay finite, and two
      // that differ do so by 2^-72 at least, so that the softmax is the same
      const float scr = fminf(fmaxf(A.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + e) << 23) * 65536.f,
                                    -0x1p100f), 0x1p100f);
      sc[0] = __shfl_sync(0xffffffffu, scr, 8 * t);
      sc[1] = __shfl_sync(0xffffffffu, scr, 8 * t + 4);
#pragma unroll
      for (int g = 0; g < G; g++) {
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < 4; x++) {
          float2 y = kv_pair16(qa[g][x], A.q.type);
          qa[g][x] = kv_pack2(y.x * up, y.y * up);
          y = __half22float2(*(const __half2*)&qa[g][x]);
          sum += y.x + y.y;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum *= -128.f / 16777216.f;
        q0[g][0] = q0[g][2] = __shfl_sync(0xffffffffu, sum, 8 * t);
        q0[g][1] = q0[g][3] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      }
    }
    float o[2 * G][4];
#pragma unroll
    for (int i = 0; i < 2 * G; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};   // heads 2t, 2t + 1; l: this thread's positions
    for (; at < stop; at++, c.pair++) {
      {
        unsigned spins = 0;
        while (!mbar_try_wait(bar + cstage, parity) && ++spins < (1u << 22)) {}
        if (__any_sync(0xffffffffu, spins >= (1u << 22))) {
          if (lane == 0) atomicOr(A.pool.err, KV_ERR_WAIT);
          kv_drain(bar, at, fetched, ST);
          gave_up = true;
          break;
        }
      }
      const uint8_t* pr = st + cstage * PB;
      // S^T: positions r and r + 8 of each record, heads 2t and 2t + 1
      float s[2][4];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const uint8_t* rec = pr + k * R::BYTES;
        uint32_t ks[2][G / 2];
        kv_lds<G / 2>(rec + R::KS + r * R::SROW, ks[0]);
        kv_lds<G / 2>(rec + R::KS + (8 + r) * R::SROW, ks[1]);
#pragma unroll
        for (int x = 0; x < 4; x++) s[k][x] = 0.f;
#pragma unroll
        for (int g = 0; g < G; g++) {
          const uint8_t* kg = rec + 8 * t + kv_kchunk<HD>(r, g);   // rows r and r + 8 have the same permutation
          const uint2 w = *(const uint2*)kg, y = *(const uint2*)(kg + 8 * HD);
          float x[4];
          kv_mma_from(x, q0[g], __byte_perm(w.x, 0u, 0x4140), __byte_perm(y.x, 0u, 0x4140), __byte_perm(w.x, 0u, 0x4342),
                      __byte_perm(y.x, 0u, 0x4342), qa[g][0], qa[g][1]);
          kv_mma(x, __byte_perm(w.y, 0u, 0x4140), __byte_perm(y.y, 0u, 0x4140), __byte_perm(w.y, 0u, 0x4342),
                 __byte_perm(y.y, 0u, 0x4342), qa[g][2], qa[g][3]);
          const __half2 d0 = *(const __half2*)&ks[0][g >> 1], d1 = *(const __half2*)&ks[1][g >> 1];
          const float f0 = (g & 1) ? __high2float(d0) : __low2float(d0), f1 = (g & 1) ? __high2float(d1) : __low2float(d1);
          s[k][0] = fmaf(x[0], f0, s[k][0]);
          s[k][1] = fmaf(x[1], f0, s[k][1]);
          s[k][2] = fmaf(x[2], f1, s[k][2]);
          s[k][3] = fmaf(x[3], f1, s[k][3]);
        }
#pragma unroll
        for (int x = 0; x < 4; x++) s[k][x] *= sc[x & 1];
      }
      const int p0 = c.pair * KV_PAIR;
      const uint32_t gone = (bad >> (2 * cstage)) & 3u;
      const bool edge = p0 < vis0 || p0 + KV_PAIR > len || gone;
      auto seen = [&](int p) { return p0 + p >= vis0 && p0 + p < len && !((gone >> (p >> 4)) & 1); };
      if (edge) {
#pragma unroll
        for (int x = 0; x < 4; x++)
          if (!seen(8 * x + r)) s[x >> 1][2 * (x & 1)] = s[x >> 1][2 * (x & 1) + 1] = -INFINITY;
      }
      float mx[2];
#pragma unroll
      for (int h = 0; h < 2; h++) mx[h] = fmaxf(fmaxf(s[0][h], s[0][2 + h]), fmaxf(s[1][h], s[1][2 + h]));
      if (__any_sync(0xffffffffu, mx[0] > m[0] + KV_SLACK || mx[1] > m[1] + KV_SLACK)) {
        float a[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], x));
          const float mn = fmaxf(m[h], mx[h]);
          a[h] = m[h] == -INFINITY ? 0.f : kv_ex2(m[h] - mn);
          m[h] = mn;
          l[h] *= a[h];
        }
#pragma unroll
        for (int i = 0; i < 2 * G; i++) {
          o[i][0] *= a[0]; o[i][1] *= a[1]; o[i][2] *= a[0]; o[i][3] *= a[1];
        }
      }
      const float mb[2] = {(m[0] == -INFINITY ? 0.f : m[0]) - KV_BOOST, (m[1] == -INFINITY ? 0.f : m[1]) - KV_BOOST};
      uint32_t pb[2][2];
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const __half2 p = __floats2half2_rn(kv_ex2(s[k][2 * j] - mb[0]), kv_ex2(s[k][2 * j + 1] - mb[1]));
          const float2 f = __half22float2(p);
          l[0] += f.x;
          l[1] += f.y;
          pb[k][j] = kv_transpose(*(const uint32_t*)&p);
        }
      // O^T += V^T P^T
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const uint8_t* rec = pr + k * R::BYTES;
        const uint8_t* vp = rec + R::V + 4 * r;
        uint32_t vs[2][G];
        kv_lds<G>(rec + R::VS + 2 * t * R::SROW, vs[0]);
        kv_lds<G>(rec + R::VS + (8 + 2 * t) * R::SROW, vs[1]);
        if (edge) {                            // a masked place's scale counts as zero (it may be NaN)
#pragma unroll
          for (int x = 0; x < 2 * G; x++) {
            const int j = x / G, y = x % G, e = y / (G / 2);
            if (!seen(16 * k + 8 * j + 2 * t + e)) vs[j][y] = 0u;
          }
        }
#pragma unroll
        for (int ch = 0; ch < R::VROW / 32; ch++) {
          uint32_t h[2][4];                    // bytes of dims 0 .. 3 as fp16 pairs (position 2t, 2t + 1), from 1024
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const uint32_t x = *(const uint32_t*)(vp + kv_vchunk<R::VROW>(2 * t + 8 * j, ch));
            const uint32_t y = *(const uint32_t*)(vp + kv_vchunk<R::VROW>(2 * t + 1 + 8 * j, ch));
            const uint32_t b0 = __byte_perm(x, y, 0x5140), b1 = __byte_perm(x, y, 0x7362);
            h[j][0] = __byte_perm(b0, 0x64646464u, 0x4140);
            h[j][1] = __byte_perm(b0, 0x64646464u, 0x4342);
            h[j][2] = __byte_perm(b1, 0x64646464u, 0x4140);
            h[j][3] = __byte_perm(b1, 0x64646464u, 0x4342);
          }
#pragma unroll
          for (int nib = 0; nib < (VB == 8 ? 1 : 2); nib++) {
            const int g = VB == 8 ? ch : 2 * ch + nib;
            uint32_t a[2][4], al[2][4];
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const uint32_t d = kv_scale_pair<G>(vs[j], g), top = FINE ? d & KV_TOP(VB) : d;
              const uint32_t low = kv_rest(d, top);
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const uint32_t code = kv_code2<VB>(h[j][e], nib);
                a[j][e] = kv_hmul2(code, top);
                if (FINE) al[j][e] = kv_hmul2(code, low);
              }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
              kv_mma(o[2 * g + e], a[0][2 * e], a[0][2 * e + 1], a[1][2 * e], a[1][2 * e + 1], pb[k][0], pb[k][1]);
              if (FINE) kv_mma(o[2 * g + e], al[0][2 * e], al[0][2 * e + 1], al[1][2 * e], al[1][2 * e + 1], pb[k][0], pb[k][1]);
            }
          }
        }
      }
      __syncwarp();                            // every lane has read the pair
      issue();
      if (++cstage == ST) {
        cstage = 0;
        parity ^= 1;
      }
    }
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], x);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], x);
    }
    if (UNIT) {                                // the warps' parts through their ring memory
      float* part = (float*)st;
#pragma unroll
      for (int g = 0; g < G; g++) {
        if (2 * t < nh)
          *(float4*)(part + (2 * t) * HD + 32 * g + 4 * r) =
              make_float4(o[2 * g][0], o[2 * g][2], o[2 * g + 1][0], o[2 * g + 1][2]);
        if (2 * t + 1 < nh)
          *(float4*)(part + (2 * t + 1) * HD + 32 * g + 4 * r) =
              make_float4(o[2 * g][1], o[2 * g][3], o[2 * g + 1][1], o[2 * g + 1][3]);
      }
      if (r == 0) {
        uml[warp][2 * t] = make_float2(m[0], l[0]);
        uml[warp][2 * t + 1] = make_float2(m[1], l[1]);
      }
      __syncthreads();
      float4* mine = (float4*)(ring + W * ST * PB);   // this CTA's sum, for the cluster
      for (int e = tid; e < nh * (HD / 4); e += NT) {
        const int h = e / (HD / 4), d = 4 * (e % (HD / 4));
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) M = fmaxf(M, uml[w][h].x);
        const float base = M == -INFINITY ? 0.f : M;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; w++) {
          const float y = kv_ex2(uml[w][h].x - base);
          const float4 v = *(const float4*)(ring + w * ST * PB + (h * HD + d) * 4);
          L += y * uml[w][h].y;
          x.x += y * v.x; x.y += y * v.y; x.z += y * v.z; x.w += y * v.w;
        }
        if (cs == 1) {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          kv_st4(A.o, (size_t)c.q * A.o.st + (size_t)(h0 + h) * A.o.sh + d,
                 make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv), vec);
        } else {
          mine[e] = x;
          if (d == 0) cml[h] = make_float2(M, L);
        }
      }
      if (cs > 1) {
        kv_cluster_sync();
        for (int e = (int)kv_cluster_rank() * NT + tid; e < nh * (HD / 4); e += cs * NT) {
          const int h = e / (HD / 4), d = 4 * (e % (HD / 4));
          float M = -INFINITY, L = 0.f;
          for (int k = 0; k < cs; k++) M = fmaxf(M, kv_ld_cluster2(kv_mapa(&cml[h], k)).x);
          const float base = M == -INFINITY ? 0.f : M;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int k = 0; k < cs; k++) {
            const float2 ml2 = kv_ld_cluster2(kv_mapa(&cml[h], k));
            const float4 v = kv_ld_cluster4(kv_mapa(&mine[e], k));
            const float y = kv_ex2(ml2.x - base);
            L += y * ml2.y;
            x.x += y * v.x; x.y += y * v.y; x.z += y * v.z; x.w += y * v.w;
          }
          const float inv = L == 0.f ? 0.f : 1.f / L;
          kv_st4(A.o, (size_t)c.q * A.o.st + (size_t)(h0 + h) * A.o.sh + d,
                 make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv), vec);
        }
        kv_cluster_sync();                       // no CTA leaves while another reads its sum
      }
      return;
    }
    if (gave_up) return;
    if (from_start && c.pair == c.end) {       // the whole unit
      const float i0 = l[0] == 0.f ? 0.f : 1.f / l[0], i1 = l[1] == 0.f ? 0.f : 1.f / l[1];
#pragma unroll
      for (int g = 0; g < G; g++) {
        const size_t off = (size_t)c.q * A.o.st + 32 * g + 4 * r;
        if (2 * t < nh)
          kv_st4(A.o, off + (size_t)(h0 + 2 * t) * A.o.sh,
                 make_float4(o[2 * g][0] * i0, o[2 * g][2] * i0, o[2 * g + 1][0] * i0, o[2 * g + 1][2] * i0), vec);
        if (2 * t + 1 < nh)
          kv_st4(A.o, off + (size_t)(h0 + 2 * t + 1) * A.o.sh,
                 make_float4(o[2 * g][1] * i1, o[2 * g][3] * i1, o[2 * g + 1][1] * i1, o[2 * g + 1][3] * i1), vec);
      }
    } else {                                   // slot 2 * share: the share begins in the unit, + 1: the unit in the share
      const int slot = 2 * share + (from_start && at > c.pair - c.beg ? 1 : 0);
      float* part = A.part + (size_t)slot * 8 * HD;
#pragma unroll
      for (int g = 0; g < G; g++) {
        if (2 * t < nh)
          *(float4*)(part + (2 * t) * HD + 32 * g + 4 * r) =
              make_float4(o[2 * g][0], o[2 * g][2], o[2 * g + 1][0], o[2 * g + 1][2]);
        if (2 * t + 1 < nh)
          *(float4*)(part + (2 * t + 1) * HD + 32 * g + 4 * r) =
              make_float4(o[2 * g][1], o[2 * g][3], o[2 * g + 1][1], o[2 * g + 1][3]);
      }
      if (r == 0) *(float4*)&ml[(size_t)slot * 8 + 2 * t] = make_float4(m[0], l[0], m[1], l[1]);
    }
    if (at < todo) {
      c.pair = c.beg;
      if (++c.u == U) locate(at, c);
    }
  }
}

// Join: one CTA per (query, head), or several with L float4s of its dims each,
// adds the partial outputs of its unit's shares; zeros where a query sees
// nothing.  L threads read one partial's row, the CTA's other thread groups
// the next partials.
// Bound by latency: one sequence of 71 MB (8 units) leaves some 220 partials a
// unit; weighing and adding them takes 8.5 us beside k_kv_token's 20, 11 with a
// CTA a head, 16 with 256 threads.  Joined by the last warp to arrive instead
// (fences and atomics), a short call took 10.1 us where the two launches take
// 8.7.
template <int HD, int L>
__global__ void __launch_bounds__(1024) k_kv_join(KvAttn A, int warps) {
  constexpr int MAXW = 4096;
  __shared__ float4 acc[1024];
  __shared__ float wgt[MAXW];                // weights of the partials (shares are at most the device's warps)
  __shared__ float red[64];
  const int tid = threadIdx.x, i = blockIdx.x, h = blockIdx.y, rows = blockDim.x / L;
  pdl_wait();
  pdl_launch();
  if (A.n_dev && i >= *A.n_dev) return;
  const long long* gpre = (const long long*)A.ml;
  const float2* ml = (const float2*)(gpre + KV_PRE);
  const int n = A.n_dev ? min(*A.n_dev, A.n) : A.n;
  const int gsz = A.heads / A.pool.kvh, HB = (gsz + 7) / 8, U = A.pool.kvh * HB;
  const int kvh = h / gsz, hh = h % gsz, u = kvh * HB + hh / 8, row = hh % 8;
  const long long p0 = gpre[i], all = gpre[i + 1] - p0, total = gpre[n];
  const long long tiles = all >> 32 ? all / U : (uint32_t)all / (uint32_t)U;
  const long long per = total >> 32 ? kv_share(total, warps) : ((uint32_t)total + warps - 1) / (uint32_t)warps;
  const int x = tid % L, y = tid / L, dim = 4 * (blockIdx.z * L + x);
  const size_t off = (size_t)i * A.o.st + (size_t)h * A.o.sh + dim;
  if (tiles == 0) {
    if (y == 0) kv_st4(A.o, off, make_float4(0.f, 0.f, 0.f, 0.f), kv_vec4(A.o));
    return;
  }
  const KvSlots S(p0 + u * tiles, tiles, per);
  if (S.cnt == 1) return;                    // finished by its warp
  float M = -INFINITY;
  float2 first = make_float2(-INFINITY, 0.f);
  for (int k = tid; k < S.cnt; k += blockDim.x) {
    const float2 e = ml[(size_t)S.slot(k) * 8 + row];
    if (k == tid) first = e;
    M = fmaxf(M, e.x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) red[tid >> 5] = M;
  __syncthreads();
  for (int w = 0; w < (int)blockDim.x / 32; w++) M = fmaxf(M, red[w]);
  const float base = M == -INFINITY ? 0.f : M;
  float l = 0.f;
  for (int k = tid; k < S.cnt; k += blockDim.x) {
    const float2 e = k == tid ? first : ml[(size_t)S.slot(k) * 8 + row];
    const float w = kv_ex2(e.x - base);
    wgt[k] = w;
    l += w * e.y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if ((tid & 31) == 0) red[32 + (tid >> 5)] = l;
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int k = y; k < S.cnt; k += rows) {
    const float4 v = *(const float4*)(A.part + ((size_t)S.slot(k) * 8 + row) * HD + dim);
    const float w = wgt[k];
    o.x += w * v.x; o.y += w * v.y; o.z += w * v.z; o.w += w * v.w;
  }
#pragma unroll
  for (int e = L; e < 32; e <<= 1) {         // a warp's rows
    o.x += __shfl_xor_sync(0xffffffffu, o.x, e);
    o.y += __shfl_xor_sync(0xffffffffu, o.y, e);
    o.z += __shfl_xor_sync(0xffffffffu, o.z, e);
    o.w += __shfl_xor_sync(0xffffffffu, o.w, e);
  }
  const int groups = L < 32 ? blockDim.x / 32 : rows;
  if (L >= 32 || (tid & 31) < L) acc[L < 32 ? (tid >> 5) * L + x : tid] = o;
  __syncthreads();
  if (y == 0) {
    l = 0.f;
    for (int w = 0; w < (int)blockDim.x / 32; w++) l += red[32 + w];
    for (int k = 1; k < groups; k++) {
      const float4 v = acc[k * L + x];
      o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    kv_st4(A.o, off, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), kv_vec4(A.o));
  }
}
