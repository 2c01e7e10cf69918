#pragma once
#include "ck_kv.cuh"
// Attention over the quantised paged cache, first form: one warp per (query
// row, head), the cached positions one after another with an online softmax
// (running maximum and sum, o rescaled when the maximum grows), all in 32
// bits.  Serves one-token and prompt queries alike.



// position and sequence of query row i; false when the row sees nothing
template <int HD, int VB>
__global__ void __launch_bounds__(128) k_kv_attn_simple(KvAttn A) {
  using R = KvRec<HD, VB>;
  constexpr int E = HD / 32;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int i = (int)(w / A.heads), h = (int)(w % A.heads);
  pdl_wait();
  pdl_launch();
  const int n_rows = A.cu ? A.rows : A.n_dev ? *A.n_dev : A.n;
  if (i >= n_rows) return;
  int seq = i, len;
  if (A.cu) {
    int lo = 0, hi = A.n;                     // last sequence whose first row is at most i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (A.cu[mid] <= i) lo = mid; else hi = mid;
    }
    seq = lo;
    len = A.len[seq] - (A.cu[seq + 1] - 1 - i);
    if (i >= A.cu[A.n]) len = 0;
  } else {
    len = A.len[i] + A.len_add;
    if (A.seq) seq = A.seq[i];
  }
  if (len > (long long)A.tab.max_blocks * A.pool.block) {
    atomicOr(A.pool.err, KV_ERR_POS);
    len = 0;
  }
  const int start = A.window > 0 && len > A.window ? len - A.window : 0;
  const int kvh = h / (A.heads / A.pool.kvh);
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const size_t off = (size_t)i * A.q.st + (size_t)h * A.q.sh + 32 * e + lane;
    q[e] = A.q.type == KV_F16 ? __half2float(((const __half*)A.q.p)[off])
                              : __bfloat162float(((const __nv_bfloat16*)A.q.p)[off]);
    o[e] = 0.f;
  }
  for (int pos = start; pos < len; pos++) {
    const uint8_t* rec = kv_record(A.pool, A.tab, seq, pos, R::BYTES, kvh);
    if (!rec) continue;
    const int p = pos & (KV_TILE - 1);
    float s = 0.f, v[E];
#pragma unroll
    for (int g = 0; g < E; g++) {
      const float kd = __half2float(*(const __half*)(rec + R::KS + (p * R::G + g) * 2));
      const float vd = __half2float(*(const __half*)(rec + R::VS + (p * R::G + g) * 2));
      s += q[g] * (((float)rec[kv_kchunk<HD>(p, g) + lane] - 128.f) * kd);
      if (VB == 8) {
        v[g] = ((float)rec[R::V + kv_vchunk<R::VROW>(p, g) + lane] - 128.f) * vd;
      } else {
        const uint32_t c = rec[R::V + kv_vchunk<R::VROW>(p, g >> 1) + lane];
        v[g] = ((float)((c >> (4 * (g & 1))) & 15u) - 8.f) * vd;
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= A.scale;
    const float mn = fmaxf(m, s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float c = expf(m - base), pr = expf(s - base);
    l = l * c + pr;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = o[e] * c + pr * v[e];
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; e++) {
    const size_t off = (size_t)i * A.o.st + (size_t)h * A.o.sh + 32 * e + lane;
    const float r = l == 0.f ? 0.f : o[e] / l;
    if (A.o.type == KV_F16) ((__half*)A.o.p)[off] = __float2half_rn(r);
    else ((__nv_bfloat16*)A.o.p)[off] = __float2bfloat16_rn(r);
  }
}
