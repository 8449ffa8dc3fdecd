// Arguments of the paged key/value cache kernels (paged_append.cu, paged_attn.cu,
// paged_attn_tc.cu) and their host launchers.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace smb {

constexpr int kPagedMaxHeads = 1024;  // query heads of one call
constexpr int kPagedMaxPage = 65536;  // tokens of a page (a power of two)
constexpr int kPagedMaxKeys = 1 << 30;  // that a row of the block table has pages for

// Bytes of one row (a head of a token) of a 4-bit cache: D/2 bytes of codes, D/32 pairs of a
// 16-bit scale and zero, rounded up to 16 bytes so that every row starts on 16 bytes.
__host__ __device__ constexpr int kv4_row_bytes(int D) { return (D / 2 + D / 8 + 15) / 16 * 16; }

// One layer's cache: rows [num_pages][kv_heads][page_size], strides in bytes (the same for
// keys and values).
struct PagedCacheArgs {
  uint8_t* k;
  uint8_t* v;
  long long num_pages;
  long long page_stride, head_stride, token_stride;
  int page_shift;  // log2 of the page size
  int Hkv;
};

struct AppendArgs {
  PagedCacheArgs c;
  const void *q, *k, *v;
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // strides in elements
  const long long* slots;
  const long long* positions;
  const double* inv_freq;  // [rot / 2] (rot = 0: no rotation)
  int rot, interleaved;
  float rope_scale, eps;
  const void *q_norm, *k_norm;  // [D] or null
  void* q_out;                  // [N, Hq, D]
  int* status;
  int N, Hq;
};

struct Kv4ReadArgs {
  const uint8_t* cache;
  long long num_pages, page_stride, head_stride, token_stride;
  int page_shift, Hkv;
  const long long* slots;
  int M;
  void* out;  // [M, Hkv, D]
};

// A segment whose keys were shared out over several CTAs, as its first CTA notes it.
struct JoinRecord {
  int last;         // last CTA with a part, -1: nothing to join
  int slot;         // slot of the first part; CTA p's is 2 p
  int head, heads;  // first query head, heads of a token
  int tok, rows;    // first row of q, rows of the tile (tokens x gs)
};

struct AttnArgs {
  PagedCacheArgs c;
  const void* q;
  long long q_ts, q_hs;  // elements
  int N, B, g;           // tokens, sequences, query heads per key head
  int gs, nsub, tq;      // heads per subgroup, subgroups per key head, tokens per row tile (tq * gs <= R)
  const int* table;
  long long table_stride;
  int max_pages;
  const int* kv_lens;
  const int* q_starts;
  const int* tree;  // null: causal
  long long tree_stride;
  int tree_words;
  float scale_log2;  // softmax scale * log2(e)
  void* out;
  long long o_ts, o_hs;
  float* lse;      // [N, Hq] or null
  int* status;     // or null
  float* part_o;   // [2 * grid][D][R] unnormalised partial outputs (rows innermost)
  float* part_ml;  // [2 * grid][R][2] their running maximum (log2 units) and sum
  JoinRecord* records;  // [grid]
  int min_tiles;        // fewest key tiles worth a CTA of its own
  int seg_cost;         // what a segment's start and end cost a CTA, in key tiles
};

cudaError_t launch_kv_append(const AppendArgs& a, int D, bool bf16, bool bits4, int sms, cudaStream_t stream, bool pdl);
cudaError_t launch_kv4_read(const Kv4ReadArgs& a, int D, bool bf16, cudaStream_t stream, bool pdl);

// What an attention call launches, a function of its sizes alone.
struct AttnPlan {
  int rows;  // R: rows of a row tile
  int grid;
  int min_tiles, seg_cost;
};
AttnPlan plan_attn_mma(int N, int B, int g, int D, bool bits4, int sms);
cudaError_t launch_attn_mma(AttnArgs a, const AttnPlan& p, int D, bool bf16, bool bits4, cudaStream_t stream, bool pdl);
// 4-bit caches and at most 8 query rows of a key head on average (false otherwise).  16 sequences of 8192
// keys, 8 key heads of 128: 72-74 us at 4 and 8 rows, 96-97 us by the kernel for 16 rows.
bool plan_attn_q4(int N, int B, int g, int D, int sms, AttnPlan* p);
cudaError_t launch_attn_q4(AttnArgs a, const AttnPlan& p, int D, bool bf16, cudaStream_t stream, bool pdl);
// tcgen05 kernel: plan_attn_tc is false for few rows and heads of 256, tc_takes for 16-bit caches with
// pages below 8 tokens.  launch_attn_tc leaves *fits false, and launches nothing, when strides do not
// make a tensor map.
// From how many query rows of a key head (on average over the sequences).  16 sequences of 8192 keys,
// 8 key heads of 128, tcgen05 against the other kernel: 16 bits 106 / 97 us at 16 rows, 106 / 115 at 24
// and 32, 107 / 199 at 48; 4 bits 165 / 153 us at 32 rows, 174 / 230 at 48.
constexpr int kTcAboveRows16 = 16, kTcAboveRows4 = 32;
bool tc_takes(const PagedCacheArgs& c, bool bits4);
bool plan_attn_tc(int N, int B, int g, int D, bool bits4, int sms, AttnPlan* p);
cudaError_t launch_attn_tc(AttnArgs a, const AttnPlan& p, int D, bool bf16, bool bits4, cudaStream_t stream, bool pdl,
                           bool* fits);
// joins the partial results of the segments that were split over CTAs
cudaError_t launch_attn_join(const AttnArgs& a, const AttnPlan& p, int D, bool bf16, cudaStream_t stream, bool pdl);

}  // namespace smb
