// Causal attention of several new tokens per sequence over the quantised
// paged cache, on tcgen05.
//
//   S = scale Q K^T,  P = exp(S - m) under the causal and window mask,
//   O = P V / sum P;  K and V = code * scale, but for fp16 outputs (FINE)
//   rounded to 16 bits (an fp16 cache's values), sums in 32 bits in tensor
//   memory.
//
// Bound by arithmetic once a sequence has some hundred tokens: per 128 x 128
// tile of scores at head_dim 128 the two products take 1024 cycles of an SM's
// tensor pipe, the exponentials 1024 of its special-function units, making K
// and V from codes about 440 issue slots of each scheduler.  So all four run
// side by side, on warps of their own:
//   1 warp    copies records (16 positions of a kv head, one bulk copy each)
//             through KvPr::STAGES staging buffers
//   4 or 8    turn codes into fp16 operand tiles of 64 positions (the same
//             arithmetic for both: V is fed to the second product as it lies,
//             its dims contiguous), K a tile ahead of V
//   2 warps   issue the products, one the scores, a tile ahead of the softmax
//             (two score buffers a query tile), one the outputs: a wait costs
//             either some 200 cycles, in which the other's products run
//   4 or 8    softmax: a thread owns a query row; it reads its 64 scores from
//             tensor memory once and writes P over them as the second
//             product's operand.  The exponentials are taken against a
//             reference maximum that is moved (and O and l rescaled) only
//             where a score passes it by 2^7, and for the first tile.  P is
//             rounded to 11 bits as the operand and kept times 2^8, so that
//             it is a normal fp16 number down to 2^-22 of the reference and
//             not lost above 2^-33; l sums the rounded P, so that the weights
//             still add up to one (0.5 % of the fresh prompts' time, below)
// A CTA holds 256 query rows (two tiles, whose products and softmaxes take
// turns; the K and V tiles serve both) or, at head_dim 256, 128.  A query row
// is a (token, head of the kv head's group) pair, so the group shares K and V.
// CTAs are numbered by depth (position of the tile within its sequence), the
// deepest first: they take longest.
//
// Measured: ragged fresh prompts of 133 GFLOP, bf16, at head_dim 128 take 192.5
// us (690 TFLOP/s, 42 % of cuBLAS's bf16 rate), the first form with one K and V
// tile and one warp for both products 296.  What bounds it now is the softmax's
// chain (scores read, maximum, exponentials, P written: some 2250 cycles for a
// K tile against both query tiles, of which the products fill 1024) and some
// 15000 cycles at a CTA's start, when Q is laid out and each role's code is
// fetched for the first time.  A part of the exponentials as polynomials on
// the FMA pipe changed nothing (188 to 193 us).
//
// Long caches with few rows would leave SMs idle: the cached positions are
// then split over several CTAs, which leave unnormalised partial rows for
// k_kv_prompt_join.
#pragma once
#include <float.h>

#include "ck_kv_attn.cuh"

#define KVP_MAXS 1024        // sequences of one launch
#define KVP_SLACK 7.f        // log2 that a score may exceed the reference maximum before O is rescaled
#define KVP_BOOST 8.f        // p is kept times 2^8 (cancelled by l): at most 2^15 as an operand, and normal down to 2^-22

// FINE: keys and values as two operand tiles each.  code * scale has 18 bits,
// and as one fp16 number loses 7 of them: 2^-12 of it, on average.  Split into
// its scale's upper bits (their product with a code is exact, KV_TOP) and the
// rest (rounded to 11 bits: 2^-14 of a key or value; 4-bit values are exact),
// the scores and the outputs are two products each.  Taken where the output is
// fp16, whose own rounding is small enough for it to show: a short prompt on
// 240 positions is off by 1.07 to 1.21 times what the same in 32 bits is, with
// one product each by up to 3.6 times, with two for the scores alone by 1.3 to
// 1.7 times; with bf16 outputs one product each is off by 1.08 times.  Time (us)
// with one and with two: fresh prompts of 133 GFLOP at head_dim 128 180 and 250
// (the scores' alone 210); the same lengths at 64 94 and 108; chunks at 256 47
// and 57, with 8-bit values 57 and 68.  Half of that is the products, the rest
// the memory of the tiles: fewer staging buffers, one V tile at head_dim 128
// (two, with two staging buffers, took 280), Q in tensor memory at 256 (in
// shared memory, with two staging buffers, 63 for 57).
template <int HD, int VB, bool FINE>
struct KvPr {
  using R = KvRec<HD, VB>;
  static constexpr int NQ = HD == 256 ? 1 : 2;            // 128-row query tiles
  static constexpr int PT = 64;                           // positions of a K / V tile
  static constexpr int BUF = HD == 256 ? 1 : 2;           // K and V tiles
  static constexpr int VBUF = FINE && HD == 128 ? 1 : BUF;
  static constexpr int SOFT = 4 * NQ, DEQ = 12 - SOFT;    // warps
  static constexpr int THREADS = (SOFT + DEQ + 3) * 32;
  static constexpr int W_COPY = SOFT + DEQ, W_S = W_COPY + 1, W_O = W_COPY + 2;   // the single warps
  static constexpr int RECS = PT / KV_TILE;
  static constexpr int STAGE_BYTES = RECS * R::BYTES;
  static constexpr int QB = 128 * HD * 2, KB = PT * HD * 2, KT = FINE ? 2 * KB : KB;
  // Q goes to tensor memory where its shared memory is wanted for K's second
  // tile (head_dim 256): it is laid out in K's place first
  static constexpr bool QT = FINE && HD == 256;
  static constexpr int SQ = 0, SK = QT ? 0 : NQ * QB, SV = SK + BUF * KT, SST = SV + VBUF * KT;
  static constexpr int FIT = (226 * 1024 - SST) / STAGE_BYTES, STAGES = FIT > 4 ? 4 : FIT;
  // at least 120 KB, so that an SM holds one CTA (each takes all of its tensor memory)
  static constexpr int NEED = SST + STAGES * STAGE_BYTES;
  static constexpr int SMEM = NEED < 120 * 1024 ? 120 * 1024 : NEED;
  static constexpr int TO = NQ * 2 * PT;                  // tensor memory: two score buffers a query tile, O, Q
  static constexpr int TQ = TO + NQ * HD;
  static_assert(TQ + (QT ? HD / 2 : 0) <= 512 && (!QT || NQ * QB <= BUF * KT), "tensor memory, and Q in K's place");
  static_assert(STAGES >= 2, "K is made a tile ahead of V");
  static_assert(SMEM <= 227 * 1024 - 1024, "shared memory");
};

// operand tile of ROWS rows, the contraction running along a row (K-major):
// core matrices of 8 rows x 16 bytes, the two halves of a 16-wide step 128
// bytes apart, 8-row groups 256, steps ROWS * 32
template <int ROWS>
__device__ __forceinline__ int kvp_kmajor(int row, int k) {
  return (k >> 4) * (ROWS * 32) + (row >> 3) * 256 + ((k >> 3) & 1) * 128 + (row & 7) * 16 + (k & 7) * 2;
}
// V: 16 bytes are 8 dims of a position; core matrices of 8 positions x 16
// bytes, 8-dim groups 128 bytes apart, 8-position groups HD * 16
template <int HD>
__device__ __forceinline__ int kvp_vmajor(int pos, int dim) {
  return (pos >> 3) * (HD * 16) + (dim >> 3) * 128 + (pos & 7) * 16 + (dim & 7) * 2;
}

__device__ __forceinline__ void umma_f16_ts(uint32_t tmem, uint32_t a, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem),
               "r"(a), "l"(db), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ float kvp_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 16 codes, neighbours in pairs, times a scale, into an operand tile
__device__ __forceinline__ void kvp_put(uint8_t* to, const uint32_t (&h)[8], uint32_t by) {
  *(uint4*)to = make_uint4(kv_hmul2(h[0], by), kv_hmul2(h[1], by), kv_hmul2(h[2], by), kv_hmul2(h[3], by));
  *(uint4*)(to + 128) = make_uint4(kv_hmul2(h[4], by), kv_hmul2(h[5], by), kv_hmul2(h[6], by), kv_hmul2(h[7], by));
}
// a plus the fp16 number h, in 32 bits
__device__ __forceinline__ void kvp_add16(float& a, unsigned short h) { asm("add.rn.f32.f16 %0, %1, %0;" : "+f"(a) : "h"(h)); }
// A value scale that is NaN, or so large that code * scale would pass fp16,
// must not meet a masked p = 0 in the second product (0 * inf): its values
// count as zero there, and the position's key becomes NaN, so that exactly the
// rows that see the position are NaN.
template <int VB>
__device__ __forceinline__ bool kvp_bad(uint32_t d) {
  return (d & 0x7fffu) > (VB == 8 ? 0x6007u : 0x6fffu);      // 515.5 (x 127) and 8188 (x 8)
}

// The first position that the token at position pos sees (pos < 0: a row
// before its sequence, which sees nothing; no sum here passes 32 bits, however
// wide the window).
__device__ __forceinline__ int kvp_low(int pos, int window) { return window > 0 && pos >= window ? pos + 1 - window : 0; }

// A whole warp waits for a phase of bar (all lanes get the same answer); gives
// up (false) after a bounded number of polls or when another role of the CTA
// has given up.
__device__ __forceinline__ bool kvp_wait(uint64_t* bar, uint32_t parity, volatile int* fail, int* err) {
  unsigned spins = 0;
  bool ok = true;
  while (!mbar_try_wait(bar, parity)) {
    if (++spins > (1u << 20)) {
      atomicOr(err, KV_ERR_WAIT);
      *fail = 1;
      ok = false;
      break;
    }
    if ((spins & 63u) == 0 && *fail) {
      ok = false;
      break;
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Whether a sequence's rows lie among the query rows.
__device__ __forceinline__ bool kvp_rows_ok(const KvAttn& A, int c0, int c1) { return c0 >= 0 && c0 <= c1 && c1 <= A.rows; }

// One warp: the rows that lie in no sequence, [0] .. [1] and [2] .. [3] of
// gaps; whether the row list goes back.  Out of line, as is kvp_zero_rows: a
// CTA's start is bound by fetching code, and with these two in its path fresh
// prompts took 193.0 us for 191.1 (190.4 without looking for such rows).
__device__ __noinline__ bool kvp_gaps(const KvAttn& A, int ends, int* gaps) {
  const int lane = threadIdx.x & 31;
  bool bad = false, back = false;
  int v0 = 0x7fffffff, v1 = -1;                // rows of the sequences that are not refused
  for (int s = lane; s < A.n; s += 32) {
    const int x = A.cu[s], y = A.cu[s + 1];
    back = back || y < x;
    if (kvp_rows_ok(A, x, y)) { v0 = min(v0, x); v1 = max(v1, y); }
    else bad = true;
  }
  bad = __any_sync(0xffffffffu, bad);
  back = __any_sync(0xffffffffu, back);
  v0 = __reduce_min_sync(0xffffffffu, v0);
  v1 = __reduce_max_sync(0xffffffffu, v1);
  const int r0 = ends & 1 ? 0 : min(max(A.cu[0], 0), A.rows), r1 = ends & 2 ? A.rows : min(max(A.cu[A.n], 0), A.rows);
  if (back || v0 > v1) v0 = v1 = r1;
  if (lane == 0) {
    gaps[0] = r0;
    gaps[1] = max(v0, r0);
    gaps[2] = v1;
    gaps[3] = max(r1, v1);
    if (bad && blockIdx.x == 0) atomicOr(A.pool.err, KV_ERR_ROWS);
  }
  return back;
}
// All CTAs, a row in turn.
__device__ __noinline__ void kvp_zero_rows(const KvAttn& A, int hd, const int* gaps) {
  const int before = gaps[1] - gaps[0], n = before + gaps[3] - gaps[2], pieces = hd / 8;
  const uint32_t zero[4] = {0u, 0u, 0u, 0u};
  const bool vec = kv_vec8(A.o);
  for (int r = blockIdx.x; r < n; r += gridDim.x) {
    const size_t row = r < before ? gaps[0] + r : gaps[2] + (r - before);
    for (int e = threadIdx.x; e < A.heads * pieces; e += blockDim.x)
      kv_put8(A.o.p, row * A.o.st + (size_t)(e / pieces) * A.o.sh + 8 * (e % pieces), zero, vec);
  }
}

// ends: 1, this launch has the call's first sequences; 2, its last.  Query rows
// that lie in no sequence are written as zeros: those before the first and after
// the last one, and those of a sequence that is refused because it leaves the
// rows; a row list that goes back is refused as a whole.
template <int HD, int VB, bool FINE>
__global__ void __launch_bounds__(KvPr<HD, VB, FINE>::THREADS, 1) k_kv_prompt(const __grid_constant__ KvAttn A, int units, int gs, int splits, int ends) {
  using C = KvPr<HD, VB, FINE>;
  using R = KvRec<HD, VB>;
  extern __shared__ __align__(1024) uint8_t sm[];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_fail;
  __shared__ int s_seq, s_tile, s_cu0, s_cu1, s_len;
  __shared__ int s_gap, s_gaps[4];             // whether rows lie in no sequence: [0] .. [1] and [2] .. [3]
  __shared__ signed char s_exp[128 * C::NQ];   // each query row's products want 2^(this - 8) times the scale
  __shared__ __align__(8) uint64_t b_full[C::STAGES], b_empty[C::STAGES], b_q, b_k[C::BUF], b_v[C::BUF], b_kf[2],
      b_s[C::NQ][2], b_p[C::NQ][2], b_pv[2], b_o, b_end, b_qt;
  __shared__ uint32_t s_miss[8];               // records of a tile that do not exist, by tile & 7 (copies run at most 5 ahead)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bt = 128 * C::NQ / gs;             // tokens of a CTA
  const int unit = blockIdx.x % units, zb = blockIdx.x / units, z = zb % splits, b = zb / splits;

  if (warp == 0) {
    // tile b, deepest first: D with f(D + 1) <= b < f(D), f(D) = tiles at depth >= D
    auto depth = [&](int c0, int c1) { return kvp_rows_ok(A, c0, c1) ? (c1 - c0 + bt - 1) / bt : 0; };
    auto odd = [&](int s, int c0, int c1) {    // refused, or rows beside it
      return !kvp_rows_ok(A, c0, c1) || (s == 0 && (ends & 1) && c0 != 0) || (s == A.n - 1 && (ends & 2) && c1 != A.rows);
    };
    // up to 32 sequences' rows stay in registers
    const bool in = lane < A.n;
    const int c0 = in ? A.cu[lane] : 0, c1 = in ? A.cu[lane + 1] : 0, ln = in ? A.len[lane] : 0;
    const int mine = depth(c0, c1);
    auto above = [&](int d) {
      int c = max(0, mine - d);
      for (int s = lane + 32; s < A.n; s += 32) c += max(0, depth(A.cu[s], A.cu[s + 1]) - d);
      return __reduce_add_sync(0xffffffffu, c);
    };
    int lo = 0, seq = -1, most = mine;         // f(lo) > b >= f(hi)
    bool gap = in && odd(lane, c0, c1), back = false;
    for (int s = lane + 32; s < A.n; s += 32) {
      most = max(most, depth(A.cu[s], A.cu[s + 1]));
      gap = gap || odd(s, A.cu[s], A.cu[s + 1]);
    }
    int hi = __reduce_max_sync(0xffffffffu, most);
    gap = __any_sync(0xffffffffu, gap);
    if (gap) back = kvp_gaps(A, ends, s_gaps);
    if (!back && above(0) > b) {
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (above(mid) > b) lo = mid; else hi = mid;
      }
      int k = b - above(lo + 1);               // the k-th sequence with more than lo tiles
      for (int s0 = 0; s0 < A.n && seq < 0; s0 += 32) {
        const int s = s0 + lane;
        const uint32_t has = __ballot_sync(0xffffffffu, (s0 == 0 ? mine : s < A.n ? depth(A.cu[s], A.cu[s + 1]) : 0) > lo);
        const int c = __popc(has);
        if (k < c) seq = s0 + __fns(has, 0, k + 1);
        k -= c;
      }
    }
    if (seq < 32 ? lane == max(seq, 0) : lane == 0) {
      s_seq = seq;
      s_tile = lo;
      s_cu0 = seq >= 32 ? A.cu[seq] : c0;
      s_cu1 = seq >= 32 ? A.cu[seq + 1] : c1;
      s_len = seq >= 32 ? A.len[seq] : ln;
      s_gap = gap;
      s_fail = 0;
    }
  } else if (warp == 1 && lane == 0) {
    for (int i = 0; i < C::STAGES; i++) {
      mbar_init(&b_full[i], 1);
      mbar_init(&b_empty[i], C::DEQ);
    }
    mbar_init(&b_q, (C::SOFT + C::DEQ) * 32);
    for (int i = 0; i < C::BUF; i++) {
      mbar_init(&b_k[i], C::DEQ * 32);
      mbar_init(&b_v[i], C::DEQ * 32);
    }
    for (int i = 0; i < 2; i++) {
      for (int w = 0; w < C::NQ; w++) {
        mbar_init(&b_s[w][i], 1);
        mbar_init(&b_p[w][i], 128);
      }
      mbar_init(&b_kf[i], 1);
      mbar_init(&b_pv[i], 1);
    }
    mbar_init(&b_o, 1);
    if (C::QT) mbar_init(&b_qt, 1);
    mbar_init(&b_end, 2);
    mbar_fence_init();
  } else if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  if (s_gap) kvp_zero_rows(A, HD, s_gaps);
  const int seq = s_seq;
  int4* desc = (int4*)A.ml + b * units + unit;      // splits: what k_kv_prompt_join joins
  if (seq < 0) {
    if (splits > 1 && z == 0 && tid == 0) *desc = make_int4(0, 0, 0, 0);
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(512));
    return;
  }
  const int n_new = s_cu1 - s_cu0, q0 = s_cu0 + s_tile * bt;
  const int ntok = min(bt, s_cu1 - q0);
  int len = max(s_len, 0);
  if (len > A.tab.max_blocks * A.pool.block) {
    if (tid == 0) atomicOr(A.pool.err, KV_ERR_POS);
    len = 0;
  }
  const int pos0 = len - n_new + s_tile * bt;  // cached position of the CTA's first token (may be negative)
  const int gsz = A.heads / A.pool.kvh, HB = (gsz + gs - 1) / gs, kvh = unit / HB;
  const int h0 = kvh * gsz + (unit % HB) * gs, nh = min(gs, gsz - (unit % HB) * gs);

  if (splits > 1 && z == 0 && tid == 0) *desc = make_int4(q0, ntok, h0, nh);

  // tiles of positions that query tile w sees: [beg, end)
  auto range = [&](int w, int& beg, int& end) {
    const int first = (128 * w) / gs, last = min(ntok, (128 * w + 127) / gs + 1) - 1;   // tokens with a row in it
    if (first > last) { beg = end = 0; return; }
    const int plo = pos0 + first, phi = pos0 + last;
    beg = kvp_low(plo, A.window) / C::PT;
    end = len > 0 && phi >= 0 ? phi / C::PT + 1 : beg;
    if (end < beg) end = beg;
  };
  int beg[C::NQ], end[C::NQ], jb = 0x7fffffff, je = 0;
#pragma unroll
  for (int w = 0; w < C::NQ; w++) {
    range(w, beg[w], end[w]);
    if (beg[w] < end[w]) { jb = min(jb, beg[w]); je = max(je, end[w]); }
  }
  if (jb > je) jb = je;
  if (splits > 1) {                            // this CTA's share of the tiles
    const int n = je - jb, a = jb + (int)((long long)n * z / splits), e = jb + (int)((long long)n * (z + 1) / splits);
    jb = a;
    je = e;
#pragma unroll
    for (int w = 0; w < C::NQ; w++) {
      beg[w] = max(beg[w], jb);
      end[w] = max(min(end[w], je), beg[w]);
    }
  }

  const uint32_t tmem = s_tmem;
  const int bpt = A.pool.block / KV_TILE;

  if (warp < C::SOFT + C::DEQ) {
    // Q in fp16, HD / 32 lanes a row, four 16-byte pieces a lane: bf16 rows are
    // brought to a power of two (as in ck_kv_attn.cuh).  The scale's sign goes
    // to q: the largest product is the largest score.  Rows go to shared memory
    // as they are, all of a warp's on their way at once, and are worked on
    // there.  (One piece a lane is bound by its chain of dependent steps, and
    // unrolled over its rows by fetching code that runs once: 12000 and 9800
    // cycles a CTA.)
    constexpr int L = HD / 32, RW = 32 / L, ROWS = 128 * C::NQ, NWQ = C::SOFT + C::DEQ;
    const bool vec = (uintptr_t)A.q.p % 16 == 0 && A.q.st % 8 == 0 && A.q.sh % 8 == 0;
    const int x = lane % L, y = lane / L;
    const uint32_t by_gs = (65536 + gs - 1) / gs;              // row / gs for rows up to 255, heads up to 128
    auto place = [&](int row, int p) { return (uint4*)(sm + C::SQ + (row >> 7) * C::QB + kvp_kmajor<128>(row & 127, 8 * (x + L * p))); };
#pragma unroll 1
    for (int row = warp * RW + y; row < ROWS; row += NWQ * RW) {
      const int tok = (row * by_gs) >> 16, head = row - tok * gs;
      const unsigned short* src = (const unsigned short*)A.q.p + (size_t)(q0 + tok) * A.q.st + (size_t)(h0 + head) * A.q.sh + 8 * x;
      const bool live = tok < ntok && head < nh;
#pragma unroll
      for (int p = 0; p < 4; p++) {
        if (!live) {
          *place(row, p) = make_uint4(0u, 0u, 0u, 0u);
        } else if (vec) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(place(row, p))), "l"(src + 8 * L * p) : "memory");
        } else {
          unsigned short* dst = (unsigned short*)place(row, p);
#pragma unroll 1
          for (int e = 0; e < 8; e++) dst[e] = src[8 * L * p + e];
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");           // each lane goes on with what it copied itself
    const uint32_t flip = A.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll 1
    for (int row = warp * RW + y; row - y < ROWS; row += NWQ * RW) {
      int e = 8;
      if (A.q.type != KV_F16 || flip) {
        uint32_t u[4][4];
#pragma unroll
        for (int p = 0; p < 4; p++) {
          const uint4 v = *place(min(row, ROWS - 1), p);
          u[p][0] = v.x; u[p][1] = v.y; u[p][2] = v.z; u[p][3] = v.w;
        }
        if (A.q.type != KV_F16) {
          uint32_t m[4];                       // the largest magnitude's bits
#pragma unroll
          for (int p = 0; p < 4; p++)
            m[p] = __vmaxu2(__vmaxu2(u[p][0] & 0x7fff7fffu, u[p][1] & 0x7fff7fffu), __vmaxu2(u[p][2] & 0x7fff7fffu, u[p][3] & 0x7fff7fffu));
          m[0] = __vmaxu2(__vmaxu2(m[0], m[1]), __vmaxu2(m[2], m[3]));
          m[0] = max(m[0] & 0xffffu, m[0] >> 16);
#pragma unroll
          for (int o = 1; o < L; o <<= 1) m[0] = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
          e = (int)(m[0] >> 7) - 127;
          e = e > 127 ? 8 : max(e, -100);
          const float up = __uint_as_float((uint32_t)(127 + 8 - e) << 23);
#pragma unroll
          for (int p = 0; p < 4; p++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              u[p][i] = kv_pack2(__uint_as_float(u[p][i] << 16) * up, __uint_as_float(u[p][i] & 0xffff0000u) * up);
        }
        if (row < ROWS)
#pragma unroll
          for (int p = 0; p < 4; p++)
            *place(row, p) = make_uint4(u[p][0] ^ flip, u[p][1] ^ flip, u[p][2] ^ flip, u[p][3] ^ flip);
      }
      if (x == 0 && row < ROWS) s_exp[row] = (signed char)e;
    }
    proxy_fence_smem();
    mbar_arrive(&b_q);
  }

  int issued = 0;                              // tiles whose copies are on their way or have landed (copy warp)
  if (warp == C::W_COPY) {
    // ---- copies: lane i fetches record i of the tile ----
    const int lowest = kvp_low(pos0, A.window);   // no row sees a position before it: its block may be another's by now
    for (int j = jb; j < je; j++, issued++) {
      const int it = j - jb, s = it % C::STAGES;
      if (it >= C::STAGES && !kvp_wait(&b_empty[s], (it / C::STAGES - 1) & 1, &s_fail, A.pool.err)) break;
      const int tile = j * C::RECS + lane;     // record of the sequence
      bool ok = lane < C::RECS && tile * KV_TILE < len && (tile + 1) * KV_TILE > lowest;
      int id = 0;
      if (ok) {
        id = A.tab.dev[(size_t)seq * A.tab.max_blocks + tile / bpt];
        ok = (unsigned)id < (unsigned)A.pool.n_blocks;
        if (!ok) atomicOr(A.pool.err, KV_ERR_BLOCK);
      }
      const uint32_t have = __ballot_sync(0xffffffffu, ok);
      uint8_t* dst = sm + C::SST + s * C::STAGE_BYTES + lane * R::BYTES;
      // a record that does not exist or is not seen: zero scales (its values
      // meet p = 0) and a mark for the softmax
      if (lane < C::RECS && !ok) {
        for (int i = R::KS; i < R::BYTES; i += 4) *(uint32_t*)(dst + i) = 0u;
        proxy_fence_smem();
      }
      if (lane == 0) s_miss[j & 7] = ~have & ((1u << C::RECS) - 1);
      __syncwarp();
      if (lane == 0) mbar_expect_tx(&b_full[s], __popc(have) * R::BYTES);
      __syncwarp();
      if (ok)
        bulk_g2s(dst, A.pool.base + (((size_t)id * A.pool.kvh + kvh) * bpt + tile % bpt) * R::BYTES, R::BYTES,
                 &b_full[s]);
    }
  } else if (warp == C::W_S || warp == C::W_O) {
    // ---- products ----
    // The whole warp runs the loop and one elected lane issues: operands that
    // the compiler sees to be the same in every lane go to the tensor core
    // from uniform registers (from a lone thread's branch each product cost
    // about 70 cycles to issue, more than it takes).
    const int n = __shfl_sync(0xffffffffu, je - jb, 0);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    int from[C::NQ], to[C::NQ];                // tiles of each query tile, counted from jb
#pragma unroll
    for (int w = 0; w < C::NQ; w++) {
      from[w] = __shfl_sync(0xffffffffu, beg[w] - jb, 0);
      to[w] = __shfl_sync(0xffffffffu, end[w] - jb, 0);
    }
    const bool leader = elect_one();
    bool ok = true;
    // descriptors: a step of 16 further along is so many 16-byte units on
    if (warp == C::W_S) {
      const uint32_t idS = (1u << 4) | ((uint32_t)(C::PT >> 3) << 17) | (8u << 24);
      const uint64_t dq = umma_desc(smem_u32(sm + C::SQ), 128, 256), dk = umma_desc(smem_u32(sm + C::SK), 128, 256);
      ok = n <= 0 || kvp_wait(&b_q, 0, &s_fail, A.pool.err);
      if (C::QT && ok && n > 0) {              // 16 of a row's elements a copy: 8 columns
        asm volatile("tcgen05.fence::after_thread_sync;");
        if (leader) {
#pragma unroll 1
          for (int k = 0; k < HD / 16; k++)
            asm volatile("tcgen05.cp.cta_group::1.128x256b [%0], %1;" ::"r"(tm + C::TQ + 8 * k), "l"(dq + k * 4096 / 16) : "memory");
          umma_commit(&b_qt);
        }
        __syncwarp();
      }
#pragma unroll 1
      for (int it = 0; ok && it < n; it++) {
        const int kb = it & (C::BUF - 1);
        ok = kvp_wait(&b_k[kb], (it / C::BUF) & 1, &s_fail, A.pool.err);
        // the score buffer: its P of two tiles ago has been multiplied
        if (it >= 2) ok = ok && kvp_wait(&b_pv[it & 1], ((it >> 1) - 1) & 1, &s_fail, A.pool.err);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;");
        if (leader) {
#pragma unroll
          for (int w = 0; w < C::NQ; w++)
            if (it >= from[w] && it < to[w]) {
#pragma unroll
              for (int k = 0; k < (FINE ? 2 : 1) * HD / 16; k++) {   // (the second tile of K follows the first)
                const uint32_t to = tm + (2 * w + (it & 1)) * C::PT;
                const uint64_t from_k = dk + kb * (C::KT / 16) + k * C::PT * 32 / 16;
                if (C::QT) umma_f16_ts(to, tm + C::TQ + 8 * (k % (HD / 16)), from_k, idS, k > 0 ? 1u : 0u);
                else umma_f16(to, dq + (w * C::QB + k % (HD / 16) * 4096) / 16, from_k, idS, k > 0 ? 1u : 0u);
              }
              umma_commit(&b_s[w][it & 1]);
            }
          umma_commit(&b_kf[it & 1]);
        }
        __syncwarp();
      }
    } else {
      const uint32_t idO = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);   // V's dims are contiguous
      const uint64_t dv = umma_desc(smem_u32(sm + C::SV), HD * 16, 128);
#pragma unroll 1
      for (int it = 0; ok && it < n; it++) {
        const int vb = it & (C::VBUF - 1);
        // two buffers: this V is announced with the next K
        if (C::BUF == 1) ok = kvp_wait(&b_v[0], it & 1, &s_fail, A.pool.err);
        else ok = kvp_wait(&b_k[(it + 1) & 1], ((it + 1) >> 1) & 1, &s_fail, A.pool.err);
#pragma unroll
        for (int w = 0; w < C::NQ; w++)
          if (ok && it >= from[w] && it < to[w]) {
            ok = kvp_wait(&b_p[w][it & 1], ((it >> 1) - ((from[w] + 1 - (it & 1)) >> 1)) & 1, &s_fail, A.pool.err);
            asm volatile("tcgen05.fence::after_thread_sync;");
            if (ok && leader) {
#pragma unroll
              for (int k = 0; k < (FINE ? 2 : 1) * C::PT / 16; k++)
                umma_f16_ts(tm + C::TO + w * HD, tm + (2 * w + (it & 1)) * C::PT + 8 * (k % (C::PT / 16)),
                            dv + vb * (C::KT / 16) + k * 2 * HD * 16 / 16, idO, it == from[w] && k == 0 ? 0u : 1u);
            }
            __syncwarp();
          }
        if (!ok) break;
        if (leader) umma_commit(&b_pv[it & 1]);
        __syncwarp();
      }
      if (leader) umma_commit(&b_o);
      __syncwarp();
    }
  } else if (warp >= C::SOFT && warp < C::SOFT + C::DEQ) {
    // ---- K and V from codes ----
    // A record's codes are cut into pieces of 8 positions x 64 dims (V in 4
    // bits: 128 dims; at head_dim 64, 16 positions): a lane takes 16 bytes of
    // codes.  A warp takes the same piece of every record (of every 2nd or 4th
    // where a record has fewer pieces than there are warps), up to 4 pieces'
    // codes in registers at a time, read before the tile they go to is free.
    // K of the next tile comes before V: the scores are wanted first.
    const int dw = warp - C::SOFT, x = lane >> 3;
    constexpr int CH = R::VROW / 32;                         // 32-byte chunks of a position's values
    constexpr int KP = HD / 32, VP = CH < 2 ? 1 : CH;        // pieces of a record
    constexpr int KW = C::DEQ / KP, VW = C::DEQ / VP;        // warps that share a piece's records
    constexpr int KN = C::RECS / KW, VN = C::RECS / VW;      // records of a warp
    constexpr int KB = KN < 4 ? KN : 4, VB4 = VN < 4 ? VN : 4;
    static_assert(KW >= 1 && VW >= 1 && KN % KB == 0 && VN % VB4 == 0, "pieces");
    const int kr = dw / KP, kp = 8 * (dw % KP & 1) + (lane & 7), kg = 2 * (dw % KP >> 1) + (x >> 1);
    const int khalf = (x & 1) ^ ((lane >> 2) & 1);           // rows 4 apart share their banks: they take the other half
    const int ksrc = kv_kchunk<HD>(kp, kg) + 16 * khalf, kscl = (kp * R::G + kg) * 2;
    const int kdst = C::SK + kvp_kmajor<C::PT>(kp, 32 * kg + 16 * khalf);
    const int vr = dw / VP, vp = CH < 2 ? 8 * (x >> 1) + (lane & 7) : 8 * (dw % VP & 1) + (lane & 7);
    const int vc = CH < 2 ? 0 : 2 * (dw % VP >> 1) + (x >> 1), vhalf = x & 1;
    const int vsrc = R::V + kv_vchunk<R::VROW>(vp, vc) + 16 * vhalf;
    const int vscl = R::VS + (vp * R::G + (VB == 8 ? vc : 2 * vc)) * 2;
    const int vdst = C::SV + kvp_vmajor<HD>(vp, (VB == 8 ? 32 * vc : 64 * vc) + 16 * vhalf);
    auto make_k = [&](int it) {
      const int s = it % C::STAGES, kb = it % C::BUF;
      const uint8_t* stg = sm + C::SST + s * C::STAGE_BYTES;
      bool ok = kvp_wait(&b_full[s], (it / C::STAGES) & 1, &s_fail, A.pool.err);
      if (!ok) return false;
#pragma unroll
      for (int k0 = 0; k0 < KN; k0 += KB) {
        uint4 c[KB];
        uint32_t d[KB];
#pragma unroll
        for (int k = 0; k < KB; k++) {
          const uint8_t* rec = stg + (kr + (k0 + k) * KW) * R::BYTES;
          c[k] = *(const uint4*)(rec + ksrc);
          d[k] = *(const unsigned short*)(rec + R::KS + kscl);
          if (kvp_bad<VB>(*(const unsigned short*)(rec + R::VS + kscl))) d[k] = 0x7fffu;
          d[k] |= d[k] << 16;
        }
        if (C::QT && k0 == 0 && it == 0) ok = kvp_wait(&b_qt, 0, &s_fail, A.pool.err);   // Q has left K's place
        if (k0 == 0 && it >= C::BUF)           // the scores of the tile that was there before are done
          ok = kvp_wait(&b_kf[(it - C::BUF) & 1], ((it - C::BUF) >> 1) & 1, &s_fail, A.pool.err);
        if (!ok) return false;
#pragma unroll
        for (int k = 0; k < KB; k++) {
          uint8_t* dst = sm + kdst + kb * C::KT + (kr + (k0 + k) * KW) * 512;
          const uint32_t w[4] = {c[k].x, c[k].y, c[k].z, c[k].w};
          const uint32_t top = FINE ? d[k] & KV_TOP(8) : d[k];
          uint32_t h[8];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            h[2 * e] = kv_half2<0x4140, 128>(w[e]);
            h[2 * e + 1] = kv_half2<0x4342, 128>(w[e]);
          }
          kvp_put(dst, h, top);
          if (FINE) kvp_put(dst + C::KB, h, kv_rest(d[k], top));
        }
      }
      proxy_fence_smem();
      // two buffers: K and the V of the tile before are announced together
      if (C::BUF == 1 || it == 0) mbar_arrive(&b_k[kb]);
      return true;
    };
    auto make_v = [&](int it) {
      const int s = it % C::STAGES, vb = it % C::VBUF, j = jb + it;
      const uint8_t* stg = sm + C::SST + s * C::STAGE_BYTES;
      bool ok = true;
#pragma unroll
      for (int k0 = 0; k0 < VN; k0 += VB4) {
        uint4 c[VB4];
        uint32_t d[VB4][2];
#pragma unroll
        for (int k = 0; k < VB4; k++) {
          const int rec = vr + (k0 + k) * VW;
          c[k] = *(const uint4*)(stg + rec * R::BYTES + vsrc);
#pragma unroll
          for (int nib = 0; nib < (VB == 8 ? 1 : 2); nib++) {
            uint32_t e = *(const unsigned short*)(stg + rec * R::BYTES + vscl + 2 * nib);
            if (kvp_bad<VB>(e) || j * C::PT + rec * KV_TILE + vp >= len) e = 0;
            d[k][nib] = e | (e << 16);
          }
        }
        if (k0 == 0 && it >= C::VBUF)          // and so is its output
          ok = kvp_wait(&b_pv[(it - C::VBUF) & 1], ((it - C::VBUF) >> 1) & 1, &s_fail, A.pool.err);
        if (!ok) return false;
#pragma unroll
        for (int k = 0; k < VB4; k++) {
          uint8_t* dst = sm + vdst + vb * C::KT + (vr + (k0 + k) * VW) * (HD * 32);
          const uint32_t w[4] = {c[k].x, c[k].y, c[k].z, c[k].w};
#pragma unroll
          for (int nib = 0; nib < (VB == 8 ? 1 : 2); nib++) {
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              h[2 * e] = kv_code2<VB>(__byte_perm(w[e], 0x64646464u, 0x4140), nib);
              h[2 * e + 1] = kv_code2<VB>(__byte_perm(w[e], 0x64646464u, 0x4342), nib);
            }
            // the other group of a 4-bit chunk: 32 dims on
            const uint32_t top = FINE ? d[k][nib] & KV_TOP(VB) : d[k][nib];
            kvp_put(dst + nib * 512, h, top);
            if (FINE) kvp_put(dst + nib * 512 + C::KB, h, kv_rest(d[k][nib], top));
          }
        }
      }
      proxy_fence_smem();
      mbar_arrive(C::BUF == 1 ? &b_v[0] : &b_k[(it + 1) & 1]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&b_empty[s]);
      return true;
    };
    bool ok = jb >= je || make_k(0);
    for (int it = 0; ok && it < je - jb; it++) {
      if (it + 1 < je - jb) ok = make_k(it + 1);
      // (nothing to announce with the last V: as a next K would, wait for the
      // scores two tiles before it, so that no warp announces twice into one
      // phase while another has not announced once)
      else if (C::BUF == 2 && it > 0) ok = kvp_wait(&b_kf[(it - 1) & 1], ((it - 1) >> 1) & 1, &s_fail, A.pool.err);
      ok = ok && make_v(it);
    }
  } else if (warp < C::SOFT) {
    // ---- softmax ----
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const int wq = warp >> 2, rl = 32 * (warp & 3) + lane;    // query tile and row of this thread
    const int rr = 128 * wq + rl, rtok = rr / gs, rhead = rr % gs;
    const bool rlive = rtok < ntok && rhead < nh;
    kvp_wait(&b_q, 0, &s_fail, A.pool.err);
    // the factor of this row's scores (a scale of 0 counts as one too small to
    // show: masked scores are -inf times it; and past 2^100 no softmax changes:
    // scores that differ do so by 2^-48 at least, the smallest product of two
    // fp16 numbers)
    const float sc = fminf(fmaxf(fabsf(A.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + s_exp[rr] - 8) << 23), 1e-37f),
                           0x1p100f);
    const int rpos = pos0 + rtok;                                 // position of the row's token
    const int rlo = kvp_low(rpos, A.window);
    // The reference before (raw) and after the factor sc (m), and less the
    // boost (mb).  wide: some lane's is so large that 32 bits round it to 2^-4
    // of an octave or worse, past 2^28 to whole ones, by which all of the row's
    // p would be off.  Such a tile's scores have the reference taken off in
    // tensor memory and are read again (less) for the exponentials: a branch
    // around the other path's registers cost all prompts 2.5 %.
    float raw = -INFINITY, m = -INFINITY, mb = -KVP_BOOST, l = 0.f;
    bool wide = false, less = false;
    const uint32_t tO = tmem + C::TO + wq * HD + lanes;
    bool ok = true;
    for (int j = beg[wq]; ok && j < end[wq];) {
      const int it = j - jb, buf = it & 1;
      // uses of this buffer by this query tile before: its tiles of the same parity
      const int use = (it >> 1) - ((beg[wq] - jb + 1 - buf) >> 1);
      const uint32_t tS = tmem + (2 * wq + buf) * C::PT + lanes;
      // visible columns: vlo .. vhi (rows of no token see all: their results go nowhere)
      const int vlo = rlive ? rlo - j * C::PT : 0, vhi = rlive ? rpos - j * C::PT : C::PT;
      ok = kvp_wait(&b_s[wq][buf], use & 1, &s_fail, A.pool.err);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;");
      const uint32_t miss = s_miss[j & 7];
      const bool edge = __any_sync(0xffffffffu, vlo > 0 || vhi < C::PT - 1 || miss != 0);
      // visible ones of the 32 columns from c on
      auto seen = [&](int c) {
        const int lo = max(vlo - c, 0), hi = min(vhi - c, 31);
        uint32_t v = lo > hi ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
        if ((miss >> (c >> 4)) & 1) v &= 0xffff0000u;
        if ((miss >> ((c >> 4) + 1)) & 1) v &= 0x0000ffffu;
        return v;
      };
      uint32_t x[64];
      tmem_ld32_nowait(tS, *(uint32_t (*)[32])&x[0]);
      tmem_ld32_nowait(tS + 32, *(uint32_t (*)[32])&x[32]);
      const uint64_t v = edge ? seen(0) | ((uint64_t)seen(32) << 32) : ~0ull;
      tmem_ld_wait(x);
      if (edge) {
#pragma unroll
        for (int e = 0; e < 64; e++)
          if (!((v >> e) & 1)) x[e] = 0xff800000u;
      }
      float mx = -INFINITY, my = -INFINITY;
#pragma unroll
      for (int e = 0; e < 64; e += 4) {
        mx = kvp_max3(mx, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
        my = kvp_max3(my, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
      }
      mx = fmaxf(mx, my);
      const float ms = mx == -INFINITY ? mx : mx * sc;
      if (!less && __any_sync(0xffffffffu, wide || ms > m + KVP_SLACK)) {   // move the reference
        const float rn = fmaxf(raw, mx), a = raw == -INFINITY ? 0.f : kv_ex2((raw - rn) * sc);
        raw = rn;
        m = rn == -INFINITY ? rn : rn * sc;
        l *= a;
        mb = (m == -INFINITY ? 0.f : m) - KVP_BOOST;
        wide = __any_sync(0xffffffffu, fabsf(mb) >= 0x1p20f);
        if (j > beg[wq]) {
          ok = kvp_wait(&b_pv[(it - 1) & 1], ((it - 1) >> 1) & 1, &s_fail, A.pool.err);   // O holds the tiles before
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            uint32_t y[32];
            tmem_ld32_nowait(tO + d, y);
            tmem_ld_wait(y);
#pragma unroll
            for (int e = 0; e < 32; e++) y[e] = __float_as_uint(__uint_as_float(y[e]) * a);
            tmem_st32(tO + d, y);
          }
        }
        if (wide) {
#pragma unroll 1
          for (int d = 0; d < C::PT; d += 32) {
            uint32_t y[32];
            tmem_ld32_nowait(tS + d, y);
            tmem_ld_wait(y);
#pragma unroll
            for (int e = 0; e < 32; e++) y[e] = __float_as_uint(__uint_as_float(y[e]) - (raw == -INFINITY ? 0.f : raw));
            tmem_st32(tS + d, y);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          mb = -KVP_BOOST;
          less = true;
          continue;
        }
      }
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      {
        const uint64_t sc2 = kv_two(sc, sc), mb2 = kv_two(-mb, -mb);
        uint32_t y[32];
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          float p, q;
          kv_split(kv_fma2(kv_two(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), sc2, mb2), p, q);
          p = kv_ex2(p);
          q = kv_ex2(q);
          y[e / 2] = kv_pack2(p, q);
          kvp_add16(sum[(e / 2 & 1) * 2], (unsigned short)y[e / 2]);   // l sums what the product takes
          kvp_add16(sum[(e / 2 & 1) * 2 + 1], (unsigned short)(y[e / 2] >> 16));
        }
        tmem_st32(tS, y);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;");
      mbar_arrive(&b_p[wq][buf]);
      less = false;
      j++;
    }
    // O / l, or this CTA's part of it
    if (ok && beg[wq] < end[wq]) ok = kvp_wait(&b_o, 0, &s_fail, A.pool.err);
    asm volatile("tcgen05.fence::after_thread_sync;");
    if (ok) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const size_t off = (size_t)(q0 + rtok) * A.o.st + (size_t)(h0 + rhead) * A.o.sh;
      const bool vec = kv_vec8(A.o);
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t x[32];
        if (beg[wq] < end[wq]) {
          tmem_ld32_nowait(tO + c, x);
          tmem_ld_wait(x);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++) x[e] = 0u;
        }
        if (splits > 1) {
          float* part = A.part + (((size_t)(b * units + unit) * splits + z) * (128 * C::NQ) + rr) * HD + c;
#pragma unroll
          for (int e = 0; e < 32; e += 4) *(uint4*)(part + e) = make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        } else if (rlive) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
              u[k] = l == 0.f ? 0u
                              : kv_to16(__uint_as_float(x[e + 2 * k]) * inv, __uint_as_float(x[e + 2 * k + 1]) * inv, A.o.type);
            kv_put8(A.o.p, off + c + e, u, vec);
          }
        }
      }
      if (splits > 1)
        ((float2*)((long long*)A.ml + KV_PRE))[((size_t)(b * units + unit) * splits + z) * (128 * C::NQ) + rr] =
            make_float2(raw == -INFINITY ? raw : fminf(fmaxf(m, -FLT_MAX), FLT_MAX), l);
    }
  }
  // no CTA leaves with a copy in flight (any role may have given up, after the
  // last copy was issued too), and none frees its tensor memory under a product
  __syncthreads();
  if (warp == C::W_COPY && s_fail) kv_drain(b_full, kv_ring_first(issued, C::STAGES), issued, C::STAGES);
  if ((warp == C::W_S || warp == C::W_O) && elect_one()) umma_commit(&b_end);
  if (warp == 2) {
    unsigned spins = 0;
    while (!mbar_try_wait(&b_end, 0) && ++spins < (1u << 20)) {}
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// Adds the parts of a split tile: one warp per query row, which loads every
// part's (m, l), then the parts' rows, whose loads are in flight together.
// Bound by latency (a few us).
template <int HD>
__global__ void __launch_bounds__(256) k_kv_prompt_join(KvAttn A, int units, int gs, int splits) {
  constexpr int ROWS = HD == 256 ? 128 : 256, E = HD / 32;
  pdl_wait();
  const int4 d = ((const int4*)A.ml)[blockIdx.x];
  const int lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5), tok = row / gs, head = row % gs;
  if (tok >= d.y || head >= d.w) return;
  const float2* ml = (const float2*)((const long long*)A.ml + KV_PRE);
  float M = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; e++) o[e] = 0.f;
  for (int z = 0; z < splits; z++) M = fmaxf(M, ml[((size_t)blockIdx.x * splits + z) * ROWS + row].x);
  const float base = M == -INFINITY ? 0.f : M;
#pragma unroll 4
  for (int z = 0; z < splits; z++) {
    const size_t at = ((size_t)blockIdx.x * splits + z) * ROWS + row;
    const float2 e = ml[at];
    const float w = kv_ex2(e.x - base);
    l += w * e.y;
#pragma unroll
    for (int i = 0; i < E; i++) o[i] += w * A.part[at * HD + 32 * i + lane];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const size_t off = (size_t)(d.x + tok) * A.o.st + (size_t)(d.z + head) * A.o.sh + lane;
#pragma unroll
  for (int i = 0; i < E; i++) {
    if (A.o.type == KV_F16) ((__half*)A.o.p)[off + 32 * i] = __float2half_rn(o[i] * inv);
    else ((__nv_bfloat16*)A.o.p)[off + 32 * i] = __float2bfloat16_rn(o[i] * inv);
  }
}
