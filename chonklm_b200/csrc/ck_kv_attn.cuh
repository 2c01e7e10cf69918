// Attention of one new token per sequence over the quantised paged cache.
//
//   s_j = scale * sum_g dk[j][g] * (q_g . ck[j][g])      (codes c, scales d per group g of 32)
//   o   = sum_j exp(s_j - m) * dv[j][g] * cv[j][g] / sum_j exp(s_j - m)
//
// Bound by the cache's bytes.  The visible 16-position records of all
// (query, kv head) units form one list, cut into equal shares, one per warp of
// the device: ragged lengths balance by themselves, one long sequence spreads
// over every SM, and no length is needed on the host.  A warp keeps KV_STAGES
// records in flight in its own part of shared memory (one cp.async.bulk each,
// completing on the warp's mbarriers); warps never wait for one another.  A
// unit that lies in one share is finished by its warp; the others leave
// unnormalised partial outputs with their (m, l), which k_kv_join adds in the
// order of the shares (no atomics: the result does not depend on timing).
//
// The up to 8 query heads of a unit share every record that is read: products
// run on m16n8k16 tensor instructions (a unit has 8 rows, too few for
// tcgen05's 64-row tiles).  S = Q K^T has the heads as rows and 8 positions as
// columns; key codes become fp16 exactly (0x6400 | byte is 1024 + byte) and
// each group's sum is multiplied by its scale in 32 bits.  O^T = V^T P^T has
// the dims as rows and the heads as columns, and S's accumulator layout is
// just P^T's operand layout, so P never leaves its registers.  Rounded to 16
// bits: p = exp(s - m) (11 bits; l sums the unrounded p) and a value
// code * scale (11 bits, as an fp16 cache would hold it).
#pragma once
#include "ck_kv.cuh"

#define KV_MAXQ 1024         // queries of one launch (their prefix sums sit in shared memory)
#define KV_SLACK 6.f         // log2 that a score may exceed the reference maximum before o is rescaled
#define KV_BOOST 8.f         // p is kept times 2^8 (cancelled by l), so that small p stay normal fp16 numbers

template <int HD, int VB>
struct KvTok {
  // 16 warps of up to 128 registers; 8 at head_dim 256, whose accumulators
  // take 64.  Stages: what fits 209 KB.
  static constexpr int WARPS = HD == 256 ? 8 : 16;
  static constexpr int STAGES = HD == 256 ? 3 : HD == 128 ? 3 : 6;
  static constexpr int SMEM = WARPS * STAGES * KvRec<HD, VB>::BYTES;
};

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
// fp16 scales of two neighbouring positions, all groups: [2][HD/32] halves
template <int W>
__device__ __forceinline__ void kv_lds(const uint8_t* p, uint32_t (&u)[W]) {
  if (W == 2) {
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

// visible records of a query: first record and their number
__device__ __forceinline__ int kv_tiles(int len, int window, int& t0) {
  const int lo = window > 0 && len > window ? len - window : 0;
  t0 = lo / KV_TILE;
  return len > 0 ? (len + KV_TILE - 1) / KV_TILE - t0 : 0;
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

template <int HD, int VB>
__global__ void __launch_bounds__(KvTok<HD, VB>::WARPS * 32, 1) k_kv_token(KvAttn A) {
  using R = KvRec<HD, VB>;
  using C = KvTok<HD, VB>;
  constexpr int G = R::G, NT = C::WARPS * 32, EPT = KV_MAXQ / NT, ST = C::STAGES;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ long long pre[KV_MAXQ + 1];
  __shared__ long long wsum[C::WARPS];
  __shared__ __align__(8) uint64_t bars[C::WARPS * ST];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gsz = A.heads / A.pool.kvh, HB = (gsz + 7) / 8, U = A.pool.kvh * HB;
  if (lane == 0)
    for (int i = 0; i < ST; i++) mbar_init(&bars[warp * ST + i], 1);
  mbar_fence_init();
  pdl_wait();
  pdl_launch();
  const int n = A.n_dev ? min(*A.n_dev, A.n) : A.n;
  {  // prefix sums of the queries' records over all their units
    long long mine[EPT], run = 0;
#pragma unroll
    for (int e = 0; e < EPT; e++) {
      const int i = tid * EPT + e;
      int t0;
      mine[e] = run;
      if (i < n) run += (long long)kv_tiles(kv_len(A, i), A.window, t0) * U;
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
    for (int e = 0; e < EPT; e++) pre[tid * EPT + e] = base + inc - run + mine[e];
    if (tid == NT - 1) pre[KV_MAXQ] = base + inc;
    __syncthreads();
  }
  long long* gpre = (long long*)A.ml;       // for k_kv_join: prefix sums, then the (m, l) pairs
  if (blockIdx.x == 0)
    for (int i = tid; i <= n; i += NT) gpre[i] = i < KV_MAXQ ? pre[i] : pre[KV_MAXQ];
  float2* ml = (float2*)(gpre + KV_MAXQ + 1);
  const long long total = pre[KV_MAXQ];
  const long long per = kv_share(total, gridDim.x * C::WARPS);
  // neighbouring shares go to different SMs, so that few records use all of them
  const int share = warp * gridDim.x + blockIdx.x;
  const long long w0 = share * per, w1 = min(total, w0 + per);
  if (w0 >= w1) return;

  uint8_t* st = ring + (size_t)warp * ST * R::BYTES;
  uint64_t* bar = &bars[warp * ST];
  const int r = lane >> 2, t = lane & 3;
  const int bpt = A.pool.block / KV_TILE;
  const bool vecq = (uintptr_t)A.q.p % 16 == 0 && A.q.st % 8 == 0 && A.q.sh % 8 == 0;

  // where a place of the list lies: query, unit of the query, record of the unit
  int fq, fu, ft, ftiles, ft0;               // the place to fetch next
  auto locate = [&](long long at, int& q, int& u, int& tile, int& tiles, int& t0) {
    int lo = 0, hi = n;                      // last query with pre[q] <= at (queries without records repeat a value)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= at) lo = mid; else hi = mid;
    }
    q = lo;
    tiles = kv_tiles(kv_len(A, q), A.window, t0);
    const long long off = at - pre[q];
    u = (int)(off / tiles);
    tile = (int)(off % tiles);
  };
  locate(w0, fq, fu, ft, ftiles, ft0);
  int cq = fq, cu = fu, ct = ft, ctiles = ftiles, ct0 = ft0;   // the place to compute next
  long long fetch = w0;
  int ids = 0, ids_at = -1;                  // block ids of 32 records from ids_at on
  uint32_t bad = 0;                          // stages whose record does not exist
  int fstage = 0;
  auto issue = [&]() {
    if (fetch >= w1) return;
    if (ids_at < 0 || ft >= ids_at + 32) {
      ids_at = ft;
      const int seq = A.seq ? A.seq[fq] : fq, tile = ft + lane;
      ids = tile < ftiles ? A.tab.dev[(size_t)seq * A.tab.max_blocks + (ft0 + tile) / bpt] : 0;
    }
    const int id = __shfl_sync(0xffffffffu, ids, ft - ids_at);
    const bool ok = (unsigned)id < (unsigned)A.pool.n_blocks;
    bad = ok ? bad & ~(1u << fstage) : bad | (1u << fstage);
    if (lane == 0) {
      if (ok) {
        mbar_expect_tx(bar + fstage, R::BYTES);
        bulk_g2s(st + fstage * R::BYTES,
                 A.pool.base + (((size_t)id * A.pool.kvh + fu / HB) * bpt + (ft0 + ft) % bpt) * R::BYTES, R::BYTES,
                 bar + fstage);
      } else {
        atomicOr(A.pool.err, KV_ERR_BLOCK);
        mbar_arrive(bar + fstage);
      }
    }
    fstage = fstage + 1 == ST ? 0 : fstage + 1;
    fetch++;
    if (++ft == ftiles) {
      ft = 0;
      ids_at = -1;
      if (++fu == U && fetch < w1) locate(fetch, fq, fu, ft, ftiles, ft0);
    }
  };
#pragma unroll
  for (int i = 0; i < ST; i++) issue();

  int cstage = 0;
  uint32_t parity = 0;
  long long at = w0;
  while (at < w1) {
    // one unit, or the part of it in this share
    const long long ubeg = at - ct, uend = ubeg + ctiles, stop = min(w1, uend);
    const int len = kv_len(A, cq), vis0 = A.window > 0 && len > A.window ? len - A.window : 0;
    const int kvh = cu / HB, h0 = kvh * gsz + (cu % HB) * 8, nh = min(8, gsz - (cu % HB) * 8);
    // Q: rows = heads, the k index in the order of the codes' bytes: thread t
    // holds dims 8t .. 8t + 7 of each group, two steps of 16
    uint32_t qa[G][4];
    float sc;
    {
      float f[G][8], top = 0.f;
#pragma unroll
      for (int g = 0; g < G; g++) {
#pragma unroll
        for (int e = 0; e < 8; e++) f[g][e] = 0.f;
        if (r < nh) {
          const unsigned short* p = (const unsigned short*)A.q.p + (size_t)cq * A.q.st + (size_t)(h0 + r) * A.q.sh + 32 * g + 8 * t;
          uint32_t x[4];
          if (vecq) {
            const uint4 v = *(const uint4*)p;
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = p[2 * e] | ((uint32_t)p[2 * e + 1] << 16);
          }
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float2 y = A.q.type == KV_F16 ? __half22float2(*(const __half2*)&x[e])
                                                : make_float2(__uint_as_float(x[e] << 16), __uint_as_float(x[e] & 0xffff0000u));
            f[g][2 * e] = y.x;
            f[g][2 * e + 1] = y.y;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(f[g][e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // a power of two brings the row's largest value to [2^8, 2^9): fp16 then
      // holds a 16-bit q of either type to within 2^-33 of that value
      int e = (int)(__float_as_uint(top) >> 23) - 127;
      e = e > 127 ? 8 : max(e, -100);
      const float up = __uint_as_float((uint32_t)(127 + 8 - e) << 23);
      sc = A.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + e - 8) << 23);
#pragma unroll
      for (int g = 0; g < G; g++)
#pragma unroll
        for (int x = 0; x < 4; x++) qa[g][x] = kv_pack2(f[g][2 * x] * up, f[g][2 * x + 1] * up);
    }
    float o[2 * G][4];
#pragma unroll
    for (int i = 0; i < 2 * G; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (; at < stop; at++, ct++) {
      {
        unsigned spins = 0;
        while (!mbar_try_wait(bar + cstage, parity)) {
          if (++spins > (1u << 22)) {
            atomicOr(A.pool.err, KV_ERR_WAIT);
            return;
          }
        }
      }
      const uint8_t* rec = st + cstage * R::BYTES;
      // S
      float s[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
      uint32_t ks[2][G];
      kv_lds<G>(rec + R::KS + 2 * t * R::SROW, ks[0]);
      kv_lds<G>(rec + R::KS + (8 + 2 * t) * R::SROW, ks[1]);
#pragma unroll
      for (int g = 0; g < G; g++) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint2 w = *(const uint2*)(rec + kv_kchunk<HD>(8 * j + r, g) + 8 * t);
          float c[4] = {0.f, 0.f, 0.f, 0.f};
          kv_mma(c, qa[g][0], 0u, qa[g][1], 0u, kv_half2<0x4140, 128>(w.x), kv_half2<0x4342, 128>(w.x));
          kv_mma(c, qa[g][2], 0u, qa[g][3], 0u, kv_half2<0x4140, 128>(w.y), kv_half2<0x4342, 128>(w.y));
          const uint32_t dp = kv_scale_pair<G>(ks[j], g);
          const float2 d = __half22float2(*(const __half2*)&dp);
          s[j][0] = fmaf(c[0], d.x, s[j][0]);
          s[j][1] = fmaf(c[1], d.y, s[j][1]);
        }
      }
      const int p0 = (ct0 + ct) * KV_TILE;
      const int lo = (bad >> cstage) & 1 ? KV_TILE : vis0 - p0, hi = len - p0;   // visible: lo <= p < hi
      const bool edge = lo > 0 || hi < KV_TILE;
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int p = 8 * j + 2 * t + e;
          s[j][e] *= sc;
          if (edge && (p < lo || p >= hi)) s[j][e] = -INFINITY;
        }
      float tm = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 1));
      tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 2));
      if (__any_sync(0xffffffffu, tm > m + KV_SLACK)) {
        const float mn = fmaxf(m, tm);
        const float a = m == -INFINITY ? 0.f : kv_ex2(m - mn);
        m = mn;
        l *= a;
        const float a0 = __shfl_sync(0xffffffffu, a, 8 * t), a1 = __shfl_sync(0xffffffffu, a, 8 * t + 4);
#pragma unroll
        for (int i = 0; i < 2 * G; i++) {
          o[i][0] *= a0; o[i][1] *= a1; o[i][2] *= a0; o[i][3] *= a1;
        }
      }
      const float mb = (m == -INFINITY ? 0.f : m) - KV_BOOST;
      uint32_t pb[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const float x = kv_ex2(s[j][0] - mb), y = kv_ex2(s[j][1] - mb);
        l += x + y;
        pb[j] = kv_pack2(x, y);
      }
      // O^T += V^T P^T
      uint32_t vs[2][G];
      kv_lds<G>(rec + R::VS + 2 * t * R::SROW, vs[0]);
      kv_lds<G>(rec + R::VS + (8 + 2 * t) * R::SROW, vs[1]);
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};   // scales of masked places count as zero (they may be NaN)
      if (edge) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int p = 8 * j + 2 * t;
          keep[j] = (p >= lo && p < hi ? 0xffffu : 0u) | (p + 1 >= lo && p + 1 < hi ? 0xffff0000u : 0u);
        }
      }
#pragma unroll
      for (int c = 0; c < R::VROW / 32; c++) {
        uint32_t w[4];
#pragma unroll
        for (int x = 0; x < 4; x++)
          w[x] = *(const uint32_t*)(rec + R::V + kv_vchunk<R::VROW>(2 * t + (x & 1) + 8 * (x >> 1), c) + 4 * r);
#pragma unroll
        for (int nib = 0; nib < (VB == 8 ? 1 : 2); nib++) {
          const int g = VB == 8 ? c : 2 * c + nib;
          uint32_t b[2][2], d[2];
#pragma unroll
          for (int j = 0; j < 2; j++) {
            uint32_t x = w[2 * j], y = w[2 * j + 1];
            if (VB == 4) {
              x = (x >> (4 * nib)) & 0x0f0f0f0fu;
              y = (y >> (4 * nib)) & 0x0f0f0f0fu;
            }
            b[j][0] = __byte_perm(x, y, 0x5140);       // dims 0, 1 of both positions
            b[j][1] = __byte_perm(x, y, 0x7362);       // dims 2, 3
            d[j] = kv_scale_pair<G>(vs[j], g) & keep[j];
          }
          constexpr int BIAS = VB == 8 ? 128 : 8;
#pragma unroll
          for (int e = 0; e < 2; e++)
            kv_mma(o[2 * g + e], kv_hmul2(kv_half2<0x4140, BIAS>(b[0][e]), d[0]),
                   kv_hmul2(kv_half2<0x4342, BIAS>(b[0][e]), d[0]), kv_hmul2(kv_half2<0x4140, BIAS>(b[1][e]), d[1]),
                   kv_hmul2(kv_half2<0x4342, BIAS>(b[1][e]), d[1]), pb[0], pb[1]);
        }
      }
      __syncwarp();                            // every lane has read the record
      issue();
      if (++cstage == ST) {
        cstage = 0;
        parity ^= 1;
      }
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (ubeg >= w0 && uend <= w1) {            // the whole unit
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float i0 = __shfl_sync(0xffffffffu, inv, 8 * t), i1 = __shfl_sync(0xffffffffu, inv, 8 * t + 4);
      const bool vec = kv_vec4(A.o);
#pragma unroll
      for (int g = 0; g < G; g++) {
        const size_t off = (size_t)cq * A.o.st + 32 * g + 4 * r;
        if (2 * t < nh)
          kv_st4(A.o, off + (size_t)(h0 + 2 * t) * A.o.sh,
                 make_float4(o[2 * g][0] * i0, o[2 * g][2] * i0, o[2 * g + 1][0] * i0, o[2 * g + 1][2] * i0), vec);
        if (2 * t + 1 < nh)
          kv_st4(A.o, off + (size_t)(h0 + 2 * t + 1) * A.o.sh,
                 make_float4(o[2 * g][1] * i1, o[2 * g][3] * i1, o[2 * g + 1][1] * i1, o[2 * g + 1][3] * i1), vec);
      }
    } else {                                   // slot 2 * share: the share's first unit, + 1: its last
      const int slot = 2 * share + (ubeg > w0 ? 1 : 0);
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
      if (t == 0) ml[(size_t)slot * 8 + r] = make_float2(m, l);
    }
    if (at < w1) {
      ct = 0;
      if (++cu == U) locate(at, cq, cu, ct, ctiles, ct0);
    }
  }
}

// Join: one CTA per (query, head) adds the partial outputs of its unit's
// shares; zeros where a query sees nothing.  HD / 4 threads read one partial's
// row (a float4 each), the CTA's other thread groups the next partials.
#define KV_JOIN_ROWS 8       // most partials read side by side
template <int HD>
__global__ void __launch_bounds__(KV_JOIN_ROWS * HD / 4) k_kv_join(KvAttn A, int warps) {
  constexpr int L = HD / 4;
  __shared__ float4 acc[KV_JOIN_ROWS][L];
  __shared__ float red[64];
  const int tid = threadIdx.x, i = blockIdx.x, h = blockIdx.y, rows = blockDim.x / L;
  pdl_wait();
  pdl_launch();
  if (A.n_dev && i >= *A.n_dev) return;
  const long long* gpre = (const long long*)A.ml;
  const float2* ml = (const float2*)(gpre + KV_MAXQ + 1);
  const int n = A.n_dev ? min(*A.n_dev, A.n) : A.n;
  const int gsz = A.heads / A.pool.kvh, HB = (gsz + 7) / 8, U = A.pool.kvh * HB;
  const int kvh = h / gsz, hh = h % gsz, u = kvh * HB + hh / 8, row = hh % 8;
  const long long p0 = gpre[i], tiles = (gpre[i + 1] - p0) / U, per = kv_share(gpre[n], warps);
  const int x = tid % L, y = tid / L;
  const size_t off = (size_t)i * A.o.st + (size_t)h * A.o.sh + 4 * x;
  if (tiles == 0) {
    if (y == 0) kv_st4(A.o, off, make_float4(0.f, 0.f, 0.f, 0.f), kv_vec4(A.o));
    return;
  }
  const long long a = p0 + u * tiles, b = a + tiles;
  const int s0 = (int)(a / per), s1 = (int)((b - 1) / per), cnt = s1 - s0 + 1;
  if (cnt == 1) return;                        // finished by its warp
  // a unit is the first one of every share it reaches into but its own first,
  // where it is that only if it begins the share
  auto slot = [&](int k) { return 2 * (s0 + k) + (k == 0 && a > s0 * per ? 1 : 0); };
  float M = -INFINITY;
  for (int k = tid; k < cnt; k += blockDim.x) M = fmaxf(M, ml[(size_t)slot(k) * 8 + row].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) red[tid >> 5] = M;
  __syncthreads();
  for (int w = 0; w < ((int)blockDim.x + 31) / 32; w++) M = fmaxf(M, red[w]);
  const float base = M == -INFINITY ? 0.f : M;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int k = y; k < cnt; k += rows) {
    const size_t s = (size_t)slot(k) * 8 + row;
    const float2 e = ml[s];
    const float4 v = *(const float4*)(A.part + s * HD + 4 * x);
    const float w = kv_ex2(e.x - base);
    l += w * e.y;
    o.x += w * v.x; o.y += w * v.y; o.z += w * v.z; o.w += w * v.w;
  }
  acc[y][x] = o;
  __syncthreads();
  if (x == 0) red[32 + y] = l;
  __syncthreads();
  if (y == 0) {
    for (int k = 1; k < rows; k++) {
      const float4 v = acc[k][x];
      o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
      l += red[32 + k];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    kv_st4(A.o, off, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), kv_vec4(A.o));
  }
}
