// Quantised paged key-value cache: what its translation unit shares with the
// engine's (kernel parameters and launch functions; no device code here).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

// error bits of a cache's device error word
#define KV_ERR_SEQ 1       // token of an unknown sequence
#define KV_ERR_POS 2       // position or length outside the block table
#define KV_ERR_BLOCK 4     // block table entry outside the pool
#define KV_ERR_WAIT 8      // a device wait gave up
#define KV_ERR_ROWS 16     // prompt: a sequence's rows leave the query rows, or go back

enum { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };

#ifdef __CUDACC__
#define KV_HD __host__ __device__
#else
#define KV_HD
#endif
// Copies through a ring of `stages` buffers, a barrier each: copy i (counted
// from 0) lies in buffer i % stages and ends phase i / stages of its barrier,
// so a wait for it asks for this parity.  (The other parity is that of the
// phase before, which has ended: asking for either waits for nothing.)
KV_HD inline unsigned kv_ring_parity(int i, int stages) { return (unsigned)(i / stages) & 1u; }
// The first copy that can still be in flight when `issued` have been issued:
// a buffer is filled again only once its copy has landed.
KV_HD inline int kv_ring_first(int issued, int stages) { return issued > stages ? issued - stages : 0; }

// One layer's pages: records of 16 positions of one kv head, [block][kv head]
// [16-position tile of the block] (record layout in ck_kv.cuh).
struct KvPool {
  uint8_t* base;
  int n_blocks, kvh, block, hd, vbits;
  int* err;
};
struct KvTable {             // block of each `block` positions of a sequence
  const int* dev;
  int n_seqs, max_blocks;
};
struct KvRows {              // [n][heads][hd], hd contiguous; strides in elements
  void* p;
  long long st, sh;
  int type;
};

struct KvStore {
  KvPool pool;
  KvTable tab;
  const int *seq, *pos;      // sequence and position of each token (seq < 0: padding, skipped)
  const int* n_dev;          // tokens, read on the device when not null
  int n, heads;              // heads 0: only k and v
  KvRows q, k, v, qo;
  const float *qw, *kw;      // norm weights or null
  const float* inv_freq;     // [hd/2]; null: no rotation
  float eps;
  int interleaved;
};

struct KvLoad {
  KvPool pool;
  KvTable tab;
  const int *seq, *pos;
  int n;
  KvRows k, v;
};

// queries of a launch of one-token attention; more take several launches, but
// not where their number is known only on the device
#define KV_MAXQ 1024

struct KvAttn {
  KvPool pool;
  KvTable tab;
  const int* seq;            // token form: table row of each query (null: query i reads row i)
  const int* len;            // cached positions of each sequence (len_add is added)
  int len_add;
  const int* n_dev;          // token form: queries, read on the device when not null (n <= KV_MAXQ then)
  const int* cu;             // prompt form: first query row of each sequence, [n + 1]
  int n;                     // token form: queries; prompt form: sequences
  int rows;                  // prompt form: query rows in all
  int heads, window;
  float scale;
  KvRows q, o;
  float *part, *ml;          // partial outputs; prefix sums and the partials' (maximum, sum)
};

// what a launch has to know of the device
struct KvDev {
  int sms;
  int clusters[4];           // clusters of 1, 2, 4 and 8 CTAs of k_kv_token by unit that run at once
};

void kv_workspace(const KvPool& p, int sms, size_t* part_bytes, size_t* ml_bytes);
cudaError_t kv_setup(const KvPool& p, int device, KvDev* d);   // kernel attributes too; not inside a stream capture
cudaError_t kv_store_launch(const KvStore& a, cudaStream_t s, bool pdl);
cudaError_t kv_load_launch(const KvLoad& a, cudaStream_t s);
cudaError_t kv_attend_launch(const KvAttn& a, const KvDev& d, cudaStream_t s, bool pdl);
cudaError_t kv_prompt_launch(const KvAttn& a, int sms, cudaStream_t s);
size_t kv_pool_bytes(const KvPool& p);

// the message of ck_global_error (defined with the engine)
int ck_global_message(int code, const char* msg);
