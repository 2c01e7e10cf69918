// Quantised paged key-value cache: record layout, the write (norms, rotation
// and quantisation in one pass) and the read back.
//
// 32 consecutive values of a head share one fp16 scale d; a value stands for
// code * d.  Keys take 8 bits, values 8 or 4:
//   8 bits: d = fp16(max |x| / 127),  code = rint(x / d) in [-127, 127]
//   4 bits: d = fp16(m / -8), m the value of the largest magnitude (the
//           positive one at a tie), code = rint(x / d) in [-8, 7]
// x / d is x * (1 / d), each rounded to 32 bits.  A group whose d rounds to
// zero has zero codes; a group with a NaN or an infinity gets d = NaN, so what
// is read from it is NaN instead of a plausible number.
//
// A record holds 16 positions of one kv head (a multiple of 128 bytes, one
// bulk copy):  key codes | value codes | key scales | value scales
//   key codes    row p of hd bytes, code + 128; the 32-byte chunk of group g
//                sits at chunk g ^ f(p)
//   value codes  8 bits: as the keys with another f; 4 bits: chunk c holds
//                groups 2c (low nibbles) and 2c + 1 (high), code + 8
//   scales       [position][hd / 32] fp16
// The chunk permutations put the 32-byte pieces that a warp of the attention
// kernels reads together (one group of several positions) into different
// shared-memory banks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "ck_kv.h"
#include "ck_ptx.cuh"

#define KV_TILE 16           // positions of a record
#define KV_GROUP 32          // values that share a scale

template <int HD, int VB>
struct KvRec {
  static constexpr int G = HD / KV_GROUP;
  static constexpr int KROW = HD, VROW = HD * VB / 8, SROW = G * 2;
  static constexpr int V = KV_TILE * KROW, KS = V + KV_TILE * VROW, VS = KS + KV_TILE * SROW;
  static constexpr int BYTES = VS + KV_TILE * SROW;
  static_assert(BYTES % 128 == 0, "records stay aligned");
};
inline int kv_record_bytes(int hd, int vb) { return KV_TILE * (hd + hd * vb / 8 + 4 * (hd / KV_GROUP)); }

// byte offset of the chunk of group g, position p (0..15), among the key codes
template <int HD>
__host__ __device__ __forceinline__ int kv_kchunk(int p, int g) {
  const int x = HD == 64 ? (p >> 1) & 1 : p & 3;
  return p * HD + ((g ^ x) << 5);
}
// the same among the value codes (c = g for 8 bits, g / 2 for 4): ROW bytes a position
template <int ROW>
__host__ __device__ __forceinline__ int kv_vchunk(int p, int c) {
  if (ROW == 32) return ((p >> 2) << 7) + (((p & 3) ^ ((p >> 2) & 1)) << 5);
  if (ROW == 64) return ((p >> 1) << 7) + (((((p & 1) << 1) | c) ^ ((p >> 1) & 3)) << 5);
  return p * ROW + ((c >> 2) << 7) + (((c & 3) ^ ((p >> 1) & 3)) << 5);
}

// Record of position pos of sequence seq, or null (with the reason in *err)
// when the table or the pool has no such place.
__device__ __forceinline__ uint8_t* kv_record(const KvPool& P, const KvTable& T, int seq, int pos, int rec_bytes,
                                              int head) {
  if ((unsigned)seq >= (unsigned)T.n_seqs) {
    atomicOr(P.err, KV_ERR_SEQ);
    return nullptr;
  }
  const int lb = 31 - __clz(P.block), slot = pos >> lb;      // blocks are powers of two
  if (pos < 0 || slot >= T.max_blocks) {
    atomicOr(P.err, KV_ERR_POS);
    return nullptr;
  }
  const int b = T.dev[(size_t)seq * T.max_blocks + slot];
  if ((unsigned)b >= (unsigned)P.n_blocks) {
    atomicOr(P.err, KV_ERR_BLOCK);
    return nullptr;
  }
  return P.base +
         ((((size_t)b * P.kvh + head) << (lb - 4)) + ((pos & (P.block - 1)) >> 4)) * (size_t)rec_bytes;
}

// Waits, a bounded time each, for the copies `from` .. `to` - 1 of a ring: a
// kernel that gives up must not leave while one of them can still write to its
// shared memory.
__device__ __forceinline__ void kv_drain(uint64_t* bar, int from, int to, int stages) {
#pragma unroll 1
  for (int i = from; i < to; i++)
    for (unsigned spins = 0; !mbar_try_wait(bar + i % stages, kv_ring_parity(i, stages)) && spins < (1u << 20); spins++) {}
}

// The upper bits of two fp16 scales, whose product with a code is exact in fp16:
// 4 bits and a 7-bit code, or 8 and one of 3 bits (or -8).
#define KV_TOP(BITS) ((BITS) == 8 ? 0xff80ff80u : 0xfff8fff8u)
// and the rest
__device__ __forceinline__ uint32_t kv_rest(uint32_t d, uint32_t top) {
  const __half2 y = __hsub2(*(const __half2*)&d, *(const __half2*)&top);
  return *(const uint32_t*)&y;
}

// ---- eight neighbouring elements of a row ----------------------------------
// they may move as 16-byte vectors: base and strides are multiples of that
__host__ __device__ inline bool kv_vec8(const KvRows& r) {
  const int n = r.type == KV_F32 ? 4 : 8;
  return (uintptr_t)r.p % 16 == 0 && r.st % n == 0 && r.sh % n == 0;
}
__host__ __device__ inline bool kv_vec4(const KvRows& r) {
  const int es = r.type == KV_F32 ? 4 : 2;
  return ((uintptr_t)r.p % (4 * es)) == 0 && r.st % 4 == 0 && r.sh % 4 == 0;
}
// two neighbouring 16-bit elements
__device__ __forceinline__ float2 kv_pair16(uint32_t x, int type) {
  return type == KV_F16 ? __half22float2(*(const __half2*)&x)
                        : make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
__device__ __forceinline__ uint32_t kv_to16(float a, float b, int type) {
  if (type == KV_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *(const uint32_t*)&h;
}
// as they lie in memory, and as numbers
template <int TYPE>
struct KvRaw8 {
  uint4 u[TYPE == KV_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* base, size_t off, bool vec) {
    constexpr int N = TYPE == KV_F32 ? 2 : 1;
    const char* p = (const char*)base + off * (TYPE == KV_F32 ? 4 : 2);
    if (vec) {
#pragma unroll
      for (int i = 0; i < N; i++) u[i] = __ldg((const uint4*)p + i);
    } else {
      uint32_t x[4 * N];
#pragma unroll
      for (int e = 0; e < 4 * N; e++)
        x[e] = TYPE == KV_F32 ? __ldg((const uint32_t*)p + e)
                              : __ldg((const unsigned short*)p + 2 * e) | ((uint32_t)__ldg((const unsigned short*)p + 2 * e + 1) << 16);
#pragma unroll
      for (int i = 0; i < N; i++) u[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
  }
  __device__ __forceinline__ void zero() {
    u[0] = make_uint4(0u, 0u, 0u, 0u);
    u[TYPE == KV_F32 ? 1 : 0] = u[0];
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t x[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
    if (TYPE == KV_F32) {
      const uint4 v = u[TYPE == KV_F32 ? 1 : 0];
#pragma unroll
      for (int e = 0; e < 4; e++) f[e] = __uint_as_float(x[e]);
      f[4] = __uint_as_float(v.x); f[5] = __uint_as_float(v.y); f[6] = __uint_as_float(v.z); f[7] = __uint_as_float(v.w);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float2 y = kv_pair16(x[e], TYPE);
        f[2 * e] = y.x;
        f[2 * e + 1] = y.y;
      }
    }
  }
};
// eight 16-bit elements
__device__ __forceinline__ void kv_put8(void* base, size_t off, const uint32_t (&u)[4], bool vec) {
  unsigned short* p = (unsigned short*)base + off;
  if (vec) {
    *(uint4*)p = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      p[2 * e] = (unsigned short)u[e];
      p[2 * e + 1] = (unsigned short)(u[e] >> 16);
    }
  }
}
__device__ __forceinline__ void kv_st4(const KvRows& r, size_t off, float4 f, bool vec) {
  const uint2 u = make_uint2(kv_to16(f.x, f.y, r.type), kv_to16(f.z, f.w, r.type));
  unsigned short* p = (unsigned short*)r.p + off;
  if (vec) {
    *(uint2*)p = u;
  } else {
    p[0] = (unsigned short)u.x; p[1] = (unsigned short)(u.x >> 16);
    p[2] = (unsigned short)u.y; p[3] = (unsigned short)(u.y >> 16);
  }
}

// ---------------------------------------------------------------------------
// Write.  `wpt` warps share a token's rows (a row is one head of q, k or v;
// rows of one kind are taken together, so a warp runs one kind's code).  A
// lane holds 8 neighbouring values of each half of a row: both members of its
// rotation pairs, with 16-byte loads and stores; a row is HD / 16 lanes, a
// group of 32 values 4 lanes.  The cosines and sines of the token's position
// are made once per warp and lie in shared memory with the norm weights, so
// that four CTAs fit an SM (three for 32-bit rows).
// Its bytes would bound it, but what does is instructions (issue slots 74 %
// busy), then latency: 16 heads and 8 kv heads of 128 take some 2500 warp
// instructions a token, two IEEE divisions a group among them, which the
// definition of scale and code needs.  Ragged prompts of 214 MB take 52 us (63 %
// of the copy bandwidth); with cosines, sines and weights in registers, three
// CTAs an SM, 69; with the same operands one by one instead of in pairs 71; five
// CTAs (48 registers) 72.  For 32-bit rows three CTAs take 69 us, two 79, four
// 73.

// two 32-bit floats at once
__device__ __forceinline__ uint64_t kv_two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void kv_split(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t kv_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t kv_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t kv_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// the larger magnitude; NaN when either is
__device__ __forceinline__ float kv_maxabs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
// codes of the lane's 8 values (4 lanes hold a group), and the group's scale.
// FOUR: 4 bits.
template <bool FOUR>
__device__ __forceinline__ uint2 kv_quant(const float (&f)[8], __half& scale) {
  float top = kv_maxabs(kv_maxabs(kv_maxabs(f[0], f[1]), kv_maxabs(f[2], f[3])),
                        kv_maxabs(kv_maxabs(f[4], f[5]), kv_maxabs(f[6], f[7])));
  top = kv_maxabs(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = kv_maxabs(top, __shfl_xor_sync(0xffffffffu, top, 2));
  float d;
  if (FOUR) {
    // the sign of the largest magnitude: positive when any value has it positive
    float up = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
    up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 1));
    up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 2));
    d = up == top ? top * -0.125f : top * 0.125f;
  } else {
    d = top / 127.f;
  }
  const bool finite = top < INFINITY;
  scale = finite ? __float2half_rn(fminf(fmaxf(d, -65504.f), 65504.f)) : __ushort_as_half(0x7fff);
  const float dd = __half2float(scale);
  const float inv = finite && dd != 0.f ? 1.f / dd : 0.f;
  // rounding by adding 1.5 * 2^23 (+ the bias): the code is the sum's low byte.
  // The lower end (and the upper one of 8 bits) is passed only where the
  // scale is so small that fp16 holds it roughly, or so large that it was cut
  float x[8];
  const uint64_t inv2 = kv_two(inv, inv), magic = kv_two(12582912.f + (FOUR ? 8.f : 128.f), 12582912.f + (FOUR ? 8.f : 128.f));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    kv_split(kv_mul2(kv_two(f[e], f[e + 1]), inv2), x[e], x[e + 1]);
    if (FOUR) x[e] = fminf(x[e], 7.f), x[e + 1] = fminf(x[e + 1], 7.f);
  }
  if (__any_sync(0xffffffffu, !(top * fabsf(inv) < (FOUR ? 8.5f : 127.5f)))) {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = fminf(fmaxf(x[e], FOUR ? -8.f : -127.f), FOUR ? 7.f : 127.f);
  }
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint64_t y = kv_add2(kv_two(x[e], x[e + 1]), magic);
    c[e] = (uint32_t)y;
    c[e + 1] = (uint32_t)(y >> 32);
  }
  return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
}

#define KV_STORE_THREADS 256
template <int HD, int VB, int TYPE>
__global__ void __launch_bounds__(KV_STORE_THREADS, TYPE == KV_F32 ? 3 : 4) k_kv_store(const __grid_constant__ KvStore A, int vec, int lw) {
  using R = KvRec<HD, VB>;
  constexpr int LPR = HD / 16, RPW = 32 / LPR, ES = TYPE == KV_F32 ? 4 : 2;   // lanes of a row, rows of a warp
  // a lane's 8 cosines, sines or weights of a half row are two 16-byte pieces:
  // first pieces of all lanes, then second ones
  __shared__ __align__(16) float cs[KV_STORE_THREADS / 32][2][HD / 2], sw[2][2][HD / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_launch();
  if (A.qw || A.kw) {
    for (int i = threadIdx.x; i < 2 * HD; i += KV_STORE_THREADS) {
      const float* w = i < HD ? A.qw : A.kw;
      const int x = i & (HD / 2 - 1);
      if (w) sw[i / HD][(i / (HD / 2)) & 1][((x >> 2) & 1) * (HD / 4) + (x >> 3) * 4 + (x & 3)] = w[i & (HD - 1)];
    }
    __syncthreads();
  }
  const int gw = blockIdx.x * (KV_STORE_THREADS / 32) + warp, wpt = 1 << lw, t = gw >> lw, sub = gw & (wpt - 1);
  if (t >= (A.n_dev ? min(*A.n_dev, A.n) : A.n)) return;
  const int lr = lane % LPR, y = lane / LPR, kvh = A.pool.kvh;

  // this warp's rounds of RPW rows: q's, then k's, then v's (those dealt out in
  // the other order, which evens out the warps' shares); each round's rows are
  // on their way while the one before is worked on
  const int step = RPW << lw, vsub = (wpt - 1 - sub) * RPW, ls = lw + (HD == 64 ? 3 : HD == 128 ? 2 : 1);
  auto rounds = [&](int rows, int first) { return first < rows ? (rows - first + step - 1) >> ls : 0; };
  const int nq = rounds(A.heads, sub * RPW), nk = nq + rounds(kvh, sub * RPW), nv = nk + rounds(kvh, vsub);
  KvRaw8<TYPE> na, nb;                           // the next round's two halves
  const char* src = nullptr;
  long long inc = 0;
  int fr = 0;                                    // and row
  auto fetch = [&](int i) {
    if (i == 0 || i == nq || i == nk) {          // the first round of a kind
      const bool isq = i < nq, isk = !isq && i < nk;
      const KvRows& m = isq ? A.q : isk ? A.k : A.v;
      fr = y + (isq || isk ? sub * RPW : vsub);
      src = (const char*)m.p + ((long long)t * m.st + (long long)fr * m.sh + 8 * lr) * ES;
      inc = step * m.sh * ES;
    } else {
      fr += step;
      src += inc;
    }
    if (i < nv && fr < (i < nq ? A.heads : kvh)) {
      const bool v = vec & (i < nq ? 1 : i < nk ? 2 : 4);
      na.load(src, 0, v);
      nb.load(src, HD / 2, v);
    } else {
      na.zero();
      nb.zero();
    }
  };
  fetch(0);
  const int seq = A.seq[t], pos = A.pos[t];
  const bool rope = A.inv_freq != nullptr, inter = A.interleaved;
  if (rope) {
    for (int i = lane; i < HD / 2; i += 32) {
      float s, c;
      sincosf((float)pos * A.inv_freq[i], &s, &c);
      const int x = inter ? i & (HD / 4 - 1) : i, at = inter ? (i / (HD / 4)) * (HD / 4) + x
                                                             : ((x >> 2) & 1) * (HD / 4) + (x >> 3) * 4 + (x & 3);
      cs[warp][0][at] = c;
      cs[warp][1][at] = s;
    }
    __syncwarp();
  }
  auto eight = [&](const float* x, uint64_t (&u)[4]) {       // the lane's of x [HD / 2], in pairs
    const ulonglong2 v = *(const ulonglong2*)(x + 4 * lr), z = *(const ulonglong2*)(x + HD / 4 + 4 * lr);
    u[0] = v.x; u[1] = v.y; u[2] = z.x; u[3] = z.y;
  };
  uint8_t* rec0 = seq >= 0 ? kv_record(A.pool, A.tab, seq, pos, R::BYTES, 0) : nullptr;   // of kv head 0
  const size_t hbytes = (size_t)(A.pool.block / KV_TILE) * R::BYTES;                      // to the next kv head's
  const int p = pos & (KV_TILE - 1), g = lr >> 2, gb = R::G / 2 + g;                      // groups of the two halves

  auto turn = [&](float (&a)[8], float (&b)[8], int key, bool norm) {   // norm and rotation
    if (norm) {
      uint64_t s2 = kv_two(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint64_t x = kv_two(a[e], a[e + 1]), z = kv_two(b[e], b[e + 1]);
        s2 = kv_fma2(z, z, kv_fma2(x, x, s2));
      }
      float ss, s1;
      kv_split(s2, ss, s1);
      ss += s1;
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss * (1.f / HD) + A.eps);
      const uint64_t inv2 = kv_two(inv, inv);
      uint64_t wa[4], wb[4];
      eight(sw[key][0], wa);
      eight(sw[key][1], wb);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        kv_split(kv_mul2(kv_mul2(kv_two(a[e], a[e + 1]), inv2), wa[e / 2]), a[e], a[e + 1]);
        kv_split(kv_mul2(kv_mul2(kv_two(b[e], b[e + 1]), inv2), wb[e / 2]), b[e], b[e + 1]);
      }
    }
    if (!rope) return;
    uint64_t c[4], n[4];
    eight(cs[warp][0], c);
    eight(cs[warp][1], n);
    if (inter) {
      float cn[8], sn[8];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        kv_split(c[e], cn[2 * e], cn[2 * e + 1]);
        kv_split(n[e], sn[2 * e], sn[2 * e + 1]);
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float x = a[e], z = a[e + 1];
        a[e] = x * cn[e / 2] - z * sn[e / 2];
        a[e + 1] = x * sn[e / 2] + z * cn[e / 2];
        x = b[e], z = b[e + 1];
        b[e] = x * cn[4 + e / 2] - z * sn[4 + e / 2];
        b[e + 1] = x * sn[4 + e / 2] + z * cn[4 + e / 2];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint64_t x = kv_two(a[e], a[e + 1]), z = kv_two(b[e], b[e + 1]);
        kv_split(kv_fma2(kv_mul2(z, n[e / 2]), kv_two(-1.f, -1.f), kv_mul2(x, c[e / 2])), a[e], a[e + 1]);
        kv_split(kv_fma2(x, n[e / 2], kv_mul2(z, c[e / 2])), b[e], b[e + 1]);
      }
    }
  };
  const bool o16 = A.qo.type == KV_F16;
  char* qo = (char*)A.qo.p + ((long long)t * A.qo.st + (long long)(y + sub * RPW) * A.qo.sh + 8 * lr) * 2;
#pragma unroll 1
  for (int i = 0; i < nv; i++) {
    float a[8], b[8];
    na.get(a);
    nb.get(b);
    const int r = fr;
    fetch(i + 1);
    if (i < nq) {
      turn(a, b, 0, A.qw != nullptr);
      if (r < A.heads) {
        uint32_t u[4], x[4];
        if (o16) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            u[e] = kv_to16(a[2 * e], a[2 * e + 1], KV_F16);
            x[e] = kv_to16(b[2 * e], b[2 * e + 1], KV_F16);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            u[e] = kv_to16(a[2 * e], a[2 * e + 1], KV_BF16);
            x[e] = kv_to16(b[2 * e], b[2 * e + 1], KV_BF16);
          }
        }
        kv_put8(qo, 0, u, vec & 8);
        kv_put8(qo, HD / 2, x, vec & 8);
      }
      qo += (long long)step * A.qo.sh * 2;
    } else if (i < nk) {
      turn(a, b, 1, A.kw != nullptr);
      __half da, db;
      const uint2 ca = kv_quant<false>(a, da), cb = kv_quant<false>(b, db);
      if (r < kvh && rec0) {
        uint8_t* rec = rec0 + r * hbytes;
        *(uint2*)(rec + kv_kchunk<HD>(p, g) + 8 * (lr & 3)) = ca;
        *(uint2*)(rec + kv_kchunk<HD>(p, gb) + 8 * (lr & 3)) = cb;
        if ((lr & 3) == 0) {
          *(__half*)(rec + R::KS + (p * R::G + g) * 2) = da;
          *(__half*)(rec + R::KS + (p * R::G + gb) * 2) = db;
        }
      }
    } else {
      __half da, db;
      uint2 ca = kv_quant<VB == 4>(a, da), cb = kv_quant<VB == 4>(b, db);
      if (VB == 4) {
        // nibbles of two neighbouring groups share a chunk: at head_dim 64 those
        // of the lane's halves, else those of lanes 4 apart (the even group's
        // lanes write them)
        if (HD == 64) {
          ca.x |= cb.x << 4;
          ca.y |= cb.y << 4;
        } else {
          ca.x |= __shfl_xor_sync(0xffffffffu, ca.x, 4) << 4;
          ca.y |= __shfl_xor_sync(0xffffffffu, ca.y, 4) << 4;
          cb.x |= __shfl_xor_sync(0xffffffffu, cb.x, 4) << 4;
          cb.y |= __shfl_xor_sync(0xffffffffu, cb.y, 4) << 4;
        }
      }
      if (r < kvh && rec0) {
        uint8_t* rec = rec0 + r * hbytes;
        if (VB == 8) {
          *(uint2*)(rec + R::V + kv_vchunk<R::VROW>(p, g) + 8 * (lr & 3)) = ca;
          *(uint2*)(rec + R::V + kv_vchunk<R::VROW>(p, gb) + 8 * (lr & 3)) = cb;
        } else if (HD == 64 || (g & 1) == 0) {
          *(uint2*)(rec + R::V + kv_vchunk<R::VROW>(p, g >> 1) + 8 * (lr & 3)) = ca;
          if (HD > 64) *(uint2*)(rec + R::V + kv_vchunk<R::VROW>(p, gb >> 1) + 8 * (lr & 3)) = cb;
        }
        if ((lr & 3) == 0) {
          *(__half*)(rec + R::VS + (p * R::G + g) * 2) = da;
          *(__half*)(rec + R::VS + (p * R::G + gb) * 2) = db;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Read back: a warp takes a token, a lane 8 neighbouring values of one of its
// heads' key and value, and KV_LOAD_ROWS heads at once, whose loads are in
// flight together.  Bound by its bytes: 293 MB in 57 us, 79 % of the copy
// bandwidth.  A row at a time, its place looked up for each, took twice the
// instructions and 68 us.

#define KV_LOAD_THREADS 256
#define KV_LOAD_ROWS 4
// eight codes (bytes) less their bias, times d, as TYPE.  For fp16 in fp16: a
// code is exact there and the product is rounded once; else in 32 bits, a byte
// u becoming a float as the bits of 2^23 + u.
template <int TYPE>
__device__ __forceinline__ void kv_out8(uint2 c, __half d, int bias, void* base, size_t off, bool vec) {
  const uint32_t w[2] = {c.x, c.y};
  if (TYPE == KV_F16) {
    uint32_t u[4];
    const __half2 b = __half2half2(__ushort_as_half((unsigned short)(0x6400 + bias))), dd = __half2half2(d);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t x = __byte_perm(w[e >> 1], 0x64646464u, (e & 1) ? 0x4342 : 0x4140);
      const __half2 y = __hmul2(__hsub2(*(const __half2*)&x, b), dd);
      u[e] = *(const uint32_t*)&y;
    }
    kv_put8(base, off, u, vec);
    return;
  }
  float f[8];
  const float fd = __half2float(d), fb = 8388608.f + bias;
#pragma unroll
  for (int e = 0; e < 8; e++)
    f[e] = (__uint_as_float(__byte_perm(w[e >> 2], 0x4b000000u, 0x7440 + (e & 3))) - fb) * fd;
  if (TYPE == KV_F32) {
    float* p = (float*)base + off;
    if (vec) {
      *(float4*)p = make_float4(f[0], f[1], f[2], f[3]);
      *((float4*)p + 1) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) p[e] = f[e];
    }
  } else {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; e++) u[e] = kv_to16(f[2 * e], f[2 * e + 1], TYPE);
    kv_put8(base, off, u, vec);
  }
}

template <int HD, int VB, int TYPE>
__global__ void __launch_bounds__(KV_LOAD_THREADS) k_kv_load(const __grid_constant__ KvLoad A, int vec) {
  using R = KvRec<HD, VB>;
  constexpr int LPR = HD / 8, RPW = 32 / LPR, ES = TYPE == KV_F32 ? 4 : 2;   // lanes of a row, rows of a warp at a time
  const int lane = threadIdx.x & 31, lr = lane % LPR, y = lane / LPR, g = lr >> 2, kvh = A.pool.kvh;
  const int t = blockIdx.x * (KV_LOAD_THREADS / 32) + (threadIdx.x >> 5);
  if (t >= A.n) return;
  const int seq = __ldg(A.seq + t), pos = __ldg(A.pos + t), p = pos & (KV_TILE - 1);
  const uint8_t* rec0 = seq >= 0 ? kv_record(A.pool, A.tab, seq, pos, R::BYTES, 0) : nullptr;
  const size_t hbytes = (size_t)(A.pool.block / KV_TILE) * R::BYTES;          // to the next kv head's record
  const int ksrc = kv_kchunk<HD>(p, g) + 8 * (lr & 3), vsrc = R::V + kv_vchunk<R::VROW>(p, VB == 8 ? g : g >> 1) + 8 * (lr & 3);
  const int dsrc = R::KS + (p * R::G + g) * 2;
  char* ko = (char*)A.k.p + ((long long)t * A.k.st + 8 * lr) * ES;
  char* vo = (char*)A.v.p + ((long long)t * A.v.st + 8 * lr) * ES;
  for (int h0 = y; h0 - y < kvh; h0 += KV_LOAD_ROWS * RPW) {
    uint2 kc[KV_LOAD_ROWS], vc[KV_LOAD_ROWS];
    __half kd[KV_LOAD_ROWS], vd[KV_LOAD_ROWS];
#pragma unroll
    for (int x = 0; x < KV_LOAD_ROWS; x++) {
      const int h = h0 + x * RPW;
      kc[x] = make_uint2(0x80808080u, 0x80808080u);           // a place that does not exist: zeros, without a sign
      vc[x] = VB == 8 ? kc[x] : make_uint2(0x88888888u, 0x88888888u);
      kd[x] = vd[x] = __ushort_as_half(0);
      if (rec0 && h < kvh) {
        const uint8_t* rec = rec0 + h * hbytes;
        kc[x] = *(const uint2*)(rec + ksrc);
        vc[x] = *(const uint2*)(rec + vsrc);
        kd[x] = *(const __half*)(rec + dsrc);
        vd[x] = *(const __half*)(rec + dsrc + (R::VS - R::KS));
      }
    }
#pragma unroll
    for (int x = 0; x < KV_LOAD_ROWS; x++) {
      const int h = h0 + x * RPW;
      if (h >= kvh) break;
      kv_out8<TYPE>(kc[x], kd[x], 128, ko + h * A.k.sh * ES, 0, vec & 1);
      if (VB == 4) {
        vc[x].x = (vc[x].x >> (4 * (g & 1))) & 0x0f0f0f0fu;
        vc[x].y = (vc[x].y >> (4 * (g & 1))) & 0x0f0f0f0fu;
      }
      kv_out8<TYPE>(vc[x], vd[x], VB == 8 ? 128 : 8, vo + h * A.v.sh * ES, 0, vec & 2);
    }
  }
}
