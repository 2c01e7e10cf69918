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
  const int slot = pos / P.block;
  if (pos < 0 || slot >= T.max_blocks) {
    atomicOr(P.err, KV_ERR_POS);
    return nullptr;
  }
  const int b = T.dev[(size_t)seq * T.max_blocks + slot];
  if ((unsigned)b >= (unsigned)P.n_blocks) {
    atomicOr(P.err, KV_ERR_BLOCK);
    return nullptr;
  }
  const int tiles = P.block / KV_TILE;
  return P.base + (((size_t)b * P.kvh + head) * tiles + (pos % P.block) / KV_TILE) * (size_t)rec_bytes;
}

// ---- four neighbouring elements of a row -----------------------------------
__device__ __forceinline__ float4 kv_ld4(const KvRows& r, size_t off, bool vec) {
  float4 f;
  if (r.type == KV_F32) {
    const float* p = (const float*)r.p + off;
    f = vec ? *(const float4*)p : make_float4(p[0], p[1], p[2], p[3]);
  } else {
    uint2 u;
    const unsigned short* p = (const unsigned short*)r.p + off;
    if (vec) u = *(const uint2*)p;
    else u = make_uint2(p[0] | ((uint32_t)p[1] << 16), p[2] | ((uint32_t)p[3] << 16));
    if (r.type == KV_F16) {
      const float2 a = __half22float2(*(const __half2*)&u.x), b = __half22float2(*(const __half2*)&u.y);
      f = make_float4(a.x, a.y, b.x, b.y);
    } else {
      f = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                      __uint_as_float(u.y & 0xffff0000u));
    }
  }
  return f;
}
__device__ __forceinline__ void kv_st4(const KvRows& r, size_t off, float4 f, bool vec) {
  if (r.type == KV_F32) {
    float* p = (float*)r.p + off;
    if (vec) *(float4*)p = f;
    else { p[0] = f.x; p[1] = f.y; p[2] = f.z; p[3] = f.w; }
    return;
  }
  uint2 u;
  if (r.type == KV_F16) {
    const __half2 a = __floats2half2_rn(f.x, f.y), b = __floats2half2_rn(f.z, f.w);
    u = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f.x, f.y), b = __floats2bfloat162_rn(f.z, f.w);
    u = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
  }
  unsigned short* p = (unsigned short*)r.p + off;
  if (vec) *(uint2*)p = u;
  else {
    p[0] = (unsigned short)u.x; p[1] = (unsigned short)(u.x >> 16);
    p[2] = (unsigned short)u.y; p[3] = (unsigned short)(u.y >> 16);
  }
}
// four elements may move as one vector: base and strides are multiples of it
__host__ __device__ inline bool kv_vec4(const KvRows& r) {
  const int es = r.type == KV_F32 ? 4 : 2;
  return ((uintptr_t)r.p % (4 * es)) == 0 && r.st % 4 == 0 && r.sh % 4 == 0;
}

// ---------------------------------------------------------------------------
// Write.  One CTA per token (blockIdx.x) and share of its rows (blockIdx.y):
// a row is one head of q, k or v.  A lane holds 4 neighbouring values (two
// such quads at head_dim 256; two rows a warp at head_dim 64), so a group is
// 8 lanes and a norm is one warp reduction.  The cosines and sines of the
// token's position are made once per CTA.

// maximum over the 8 lanes of a group
__device__ __forceinline__ uint32_t group_umax(uint32_t v) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ uint32_t kv_abs4(const float4& f) {
  return max(max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu),
             max(__float_as_uint(f.z) & 0x7fffffffu, __float_as_uint(f.w) & 0x7fffffffu));
}
__device__ __forceinline__ uint32_t kv_code(float x, float inv, float lo, float hi, int bias) {
  return (uint32_t)(__float2int_rn(fminf(fmaxf(x * inv, lo), hi)) + bias);
}
__device__ __forceinline__ uint32_t kv_pack(const float4& f, float inv, float lo, float hi, int bias) {
  return kv_code(f.x, inv, lo, hi, bias) | (kv_code(f.y, inv, lo, hi, bias) << 8) |
         (kv_code(f.z, inv, lo, hi, bias) << 16) | (kv_code(f.w, inv, lo, hi, bias) << 24);
}
// scale of the lane's group and its reciprocal (0 where the codes are zero)
__device__ __forceinline__ __half kv_scale(const float4& f, bool four, float& inv) {
  const uint32_t top = group_umax(kv_abs4(f));
  float d;
  if (four) {
    // the sign of the largest magnitude: positive when any value has it positive
    const float m = __uint_as_float(top);
    const uint32_t pos = group_umax((f.x == m || f.y == m || f.z == m || f.w == m) ? 1u : 0u);
    d = (pos ? m : -m) / -8.f;
  } else {
    d = __uint_as_float(top) / 127.f;
  }
  d = fminf(fmaxf(d, -65504.f), 65504.f);
  const __half h = top >= 0x7f800000u ? __ushort_as_half(0x7fff) : __float2half_rn(d);
  const float dd = __half2float(h);
  inv = (top >= 0x7f800000u || dd == 0.f) ? 0.f : 1.f / dd;
  return h;
}

#define KV_STORE_THREADS 256
template <int HD>
__global__ void __launch_bounds__(KV_STORE_THREADS) k_kv_store(KvStore A, int vec) {
  constexpr int LPR = HD == 64 ? 16 : 32;    // lanes of a row
  constexpr int RPW = 32 / LPR;              // rows of a warp
  constexpr int NQ = HD / (4 * LPR);         // quads of a lane
  constexpr int NW = KV_STORE_THREADS / 32;
  __shared__ float2 cs[HD / 2];
  const int t = blockIdx.x;
  pdl_wait();
  pdl_launch();
  if (A.n_dev && t >= *A.n_dev) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seq = A.seq[t], pos = A.pos[t] + A.pos_add;
  if (A.inv_freq) {
    if (tid < HD / 2) {
      float sn, cn;
      sincosf((float)pos * A.inv_freq[tid], &sn, &cn);
      cs[tid] = make_float2(cn, sn);
    }
    __syncthreads();
  }
  const int kvh = A.pool.kvh, H = A.heads, rows = H + 2 * kvh;
  const int rec_bytes = KV_TILE * (HD + HD * A.pool.vbits / 8 + 4 * (HD / KV_GROUP));
  const int lr = lane & (LPR - 1);
  const bool vq = vec & 1, vk = vec & 2, vv = vec & 4, vo = vec & 8;
  for (int r0 = (blockIdx.y * NW + warp) * RPW; r0 < rows; r0 += gridDim.y * NW * RPW) {
    const int r = r0 + lane / LPR;
    const bool live = r < rows;
    const int kind = r < H ? 0 : r < H + kvh ? 1 : 2;      // q, k, v
    const int head = kind == 0 ? r : kind == 1 ? r - H : r - H - kvh;
    float4 f[NQ];
#pragma unroll
    for (int j = 0; j < NQ; j++) {
      f[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (live) {
        const KvRows& src = kind == 0 ? A.q : kind == 1 ? A.k : A.v;
        f[j] = kv_ld4(src, (size_t)t * src.st + (size_t)head * src.sh + 128 * j + 4 * lr,
                      kind == 0 ? vq : kind == 1 ? vk : vv);
      }
    }
    const float* w = kind == 0 ? A.qw : A.kw;
    if (A.qw || A.kw) {      // the reduction's shuffles need the whole warp
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < NQ; j++) ss += f[j].x * f[j].x + f[j].y * f[j].y + f[j].z * f[j].z + f[j].w * f[j].w;
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (kind < 2 && w) {
        const float inv = 1.0f / sqrtf(ss / (float)HD + A.eps);
#pragma unroll
        for (int j = 0; j < NQ; j++) {
          const float* wj = w + 128 * j + 4 * lr;
          f[j].x = (f[j].x * inv) * wj[0];
          f[j].y = (f[j].y * inv) * wj[1];
          f[j].z = (f[j].z * inv) * wj[2];
          f[j].w = (f[j].w * inv) * wj[3];
        }
      }
    }
    if (A.inv_freq) {
      if (A.interleaved) {
#pragma unroll
        for (int j = 0; j < NQ; j++) {
          const float2 c0 = cs[64 * j + 2 * lr], c1 = cs[64 * j + 2 * lr + 1];
          const float4 x = f[j];
          if (kind < 2)
            f[j] = make_float4(x.x * c0.x - x.y * c0.y, x.x * c0.y + x.y * c0.x, x.z * c1.x - x.w * c1.y,
                               x.z * c1.y + x.w * c1.x);
        }
      } else if (NQ == 2) {   // dims d and d + 128 sit in one lane
        float* a = (float*)&f[0];
        float* b = (float*)&f[NQ - 1];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 c = cs[4 * lr + e];
          const float x = a[e], y = b[e];
          if (kind < 2) {
            a[e] = x * c.x - y * c.y;
            b[e] = x * c.y + y * c.x;
          }
        }
      } else {                // dims d and d + hd/2 sit half a row apart
        const bool up = lr >= LPR / 2;
        float* a = (float*)&f[0];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 c = cs[(4 * lr + e) & (HD / 2 - 1)];
          const float o = __shfl_xor_sync(0xffffffffu, a[e], LPR / 2);
          if (kind < 2) a[e] = up ? o * c.y + a[e] * c.x : a[e] * c.x - o * c.y;
        }
      }
    }
    // quantisation is computed by every lane (its shuffles need the whole
    // warp); q rows only ignore it
    const bool four = kind == 2 && A.pool.vbits == 4;
    uint8_t* rec = nullptr;
    if (live && kind > 0 && seq >= 0) rec = kv_record(A.pool, A.tab, seq, pos, rec_bytes, head);
    const int p = pos & (KV_TILE - 1);
    const int vrow = HD * A.pool.vbits / 8;
#pragma unroll
    for (int j = 0; j < NQ; j++) {
      const int g = 4 * j + lr / 8;          // group of this lane's quad
      float inv;
      const __half d = kv_scale(f[j], four, inv);
      const uint32_t c8 = kv_pack(f[j], inv, four ? -8.f : -127.f, four ? 7.f : 127.f, four ? 8 : 128);
      const uint32_t other = __shfl_xor_sync(0xffffffffu, c8, 8);   // the neighbouring group's codes (4 bits)
      if (live && kind == 0 && A.qo.p)
        kv_st4(A.qo, (size_t)t * A.qo.st + (size_t)head * A.qo.sh + 128 * j + 4 * lr, f[j], vo);
      if (rec) {
        const int vs = KV_TILE * (HD + vrow) + (kind == 2 ? KV_TILE * 2 * (HD / KV_GROUP) : 0);
        if ((lr & 7) == 0) *(__half*)(rec + vs + (p * (HD / KV_GROUP) + g) * 2) = d;
        if (kind == 1) {
          *(uint32_t*)(rec + kv_kchunk<HD>(p, g) + 4 * (lr & 7)) = c8;
        } else if (!four) {
          *(uint32_t*)(rec + KV_TILE * HD + kv_vchunk<HD>(p, g) + 4 * (lr & 7)) = c8;
        } else if ((g & 1) == 0) {
          *(uint32_t*)(rec + KV_TILE * HD + kv_vchunk<HD / 2>(p, g >> 1) + 4 * (lr & 7)) = c8 | (other << 4);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Read back: a warp takes (token, kv head) rows, a lane 4 neighbouring values
// of the key and of the value.

#define KV_LOAD_THREADS 256
template <int HD, int VB>
__global__ void __launch_bounds__(KV_LOAD_THREADS) k_kv_load(KvLoad A, int vec) {
  using R = KvRec<HD, VB>;
  constexpr int Q = HD / 4;                  // lanes of a row
  const long long i = (long long)blockIdx.x * KV_LOAD_THREADS + threadIdx.x;
  const long long row = i / Q;
  if (row >= (long long)A.n * A.pool.kvh) return;
  const int lr = (int)(i % Q), t = (int)(row / A.pool.kvh), head = (int)(row % A.pool.kvh);
  const int seq = A.seq[t], pos = A.pos[t];
  float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
  const uint8_t* rec = seq >= 0 ? kv_record(A.pool, A.tab, seq, pos, R::BYTES, head) : nullptr;
  if (rec) {
    const int p = pos & (KV_TILE - 1), g = lr >> 3;
    const uint32_t kc = *(const uint32_t*)(rec + kv_kchunk<HD>(p, g) + 4 * (lr & 7));
    const float kd = __half2float(*(const __half*)(rec + R::KS + (p * R::G + g) * 2));
    uint32_t vc = *(const uint32_t*)(rec + R::V + kv_vchunk<R::VROW>(p, VB == 8 ? g : g >> 1) + 4 * (lr & 7));
    const float vd = __half2float(*(const __half*)(rec + R::VS + (p * R::G + g) * 2));
    if (VB == 4) vc = (vc >> (4 * (g & 1))) & 0x0f0f0f0fu;
    const float vb = VB == 8 ? 128.f : 8.f;
    k = make_float4(((float)(kc & 255u) - 128.f) * kd, ((float)((kc >> 8) & 255u) - 128.f) * kd,
                    ((float)((kc >> 16) & 255u) - 128.f) * kd, ((float)(kc >> 24) - 128.f) * kd);
    v = make_float4(((float)(vc & 255u) - vb) * vd, ((float)((vc >> 8) & 255u) - vb) * vd,
                    ((float)((vc >> 16) & 255u) - vb) * vd, ((float)(vc >> 24) - vb) * vd);
  }
  kv_st4(A.k, (size_t)t * A.k.st + (size_t)head * A.k.sh + 4 * lr, k, vec & 1);
  kv_st4(A.v, (size_t)t * A.v.st + (size_t)head * A.v.sh + 4 * lr, v, vec & 2);
}
