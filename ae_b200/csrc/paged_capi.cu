// C ABI entry points of the paged key/value cache: argument checks and launches.
#include <algorithm>

#include "../../include/ae_b200.h"
#include "host.h"
#include "paged.h"

using namespace smb;

namespace {

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool storage(int dtype) { return dtype == SMB_DTYPE_F16 || dtype == SMB_DTYPE_BF16; }

int cache_args(const smb_paged_cache_t* c, PagedCacheArgs* out) {
  if (c == nullptr) return SMB_ERR_NULL;
  if (c->bits != 16 && c->bits != 4) return SMB_ERR_DTYPE;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return SMB_ERR_SHAPE;
  if (c->kv_heads < 1 || c->kv_heads > kPagedMaxHeads || c->num_pages < 0) return SMB_ERR_SHAPE;
  if (c->page_size < 1 || c->page_size > kPagedMaxPage || (c->page_size & (c->page_size - 1)) != 0) return SMB_ERR_SHAPE;
  if (c->page_stride < 0 || c->head_stride < 0 || c->token_stride < 0) return SMB_ERR_SHAPE;
  if (c->page_stride % 16 || c->head_stride % 16 || c->token_stride % 16) return SMB_ERR_ALIGN;
  if (!aligned16(c->k) || !aligned16(c->v)) return SMB_ERR_ALIGN;
  if (c->num_pages > 0 && (c->k == nullptr || c->v == nullptr)) return SMB_ERR_NULL;
  out->k = static_cast<uint8_t*>(c->k);
  out->v = static_cast<uint8_t*>(c->v);
  out->num_pages = c->num_pages;
  out->page_stride = c->page_stride;
  out->head_stride = c->head_stride;
  out->token_stride = c->token_stride;
  out->page_shift = __builtin_ctz(static_cast<unsigned>(c->page_size));
  out->Hkv = c->kv_heads;
  return SMB_OK;
}

int need_b200(DeviceInfo* di) {
  const int rc = device_info(di);
  if (rc != SMB_OK) return rc;
  return di->sm100 ? SMB_OK : SMB_ERR_ARCH;
}

int done(cudaError_t err) { return err == cudaSuccess ? SMB_OK : cuda_fail(err); }

// Sizes of an attention call, checked.
int attn_sizes(int N, int B, int Hq, int Hkv, int D, int bits) {
  if (D != 64 && D != 128 && D != 256) return SMB_ERR_SHAPE;
  if (bits != 16 && bits != 4) return SMB_ERR_DTYPE;
  if (N < 0 || B < 0 || Hkv < 1 || Hq < Hkv || Hq % Hkv != 0 || Hq > kPagedMaxHeads) return SMB_ERR_SHAPE;
  if (static_cast<long long>(N) * Hq > 0x7fffffffll) return SMB_ERR_SHAPE;
  return SMB_OK;
}

size_t attn_ws(const AttnPlan& p, int D) {
  return static_cast<size_t>(2) * p.grid * p.rows * (D + 2) * sizeof(float) + p.grid * sizeof(JoinRecord);
}

}  // namespace

extern "C" {

int smb_kv4_row_bytes(int head_dim) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return SMB_ERR_SHAPE;
  return kv4_row_bytes(head_dim);
}

int smb_kv_append(const smb_append_args_t* p, smb_stream_t stream) {
  if (p == nullptr) return SMB_ERR_NULL;
  if (p->struct_bytes != sizeof(*p)) return SMB_ERR_SHAPE;
  AppendArgs a{};
  int rc = cache_args(&p->cache, &a.c);
  if (rc != SMB_OK) return rc;
  if (!storage(p->dtype)) return SMB_ERR_DTYPE;
  const int D = p->cache.head_dim, N = p->N, Hq = p->Hq, rot = p->rot;
  if (N < 0 || Hq < 1 || Hq > kPagedMaxHeads || rot < 0 || rot > D || rot % 16 != 0) return SMB_ERR_SHAPE;
  if (N == 0) return SMB_OK;
  if (p->q == nullptr || p->k == nullptr || p->v == nullptr || p->slots == nullptr || p->q_out == nullptr)
    return SMB_ERR_NULL;
  if (rot > 0 && (p->positions == nullptr || p->inv_freq == nullptr)) return SMB_ERR_NULL;
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) || !aligned16(p->q_out) || !aligned16(p->q_norm) ||
      !aligned16(p->k_norm))
    return SMB_ERR_ALIGN;
  if (p->q_out == p->q) return SMB_ERR_ALIGN;
  for (int i = 0; i < 2; ++i)
    if (p->q_strides[i] % 8 != 0 || p->k_strides[i] % 8 != 0 || p->v_strides[i] % 8 != 0) return SMB_ERR_ALIGN;
  DeviceInfo di;
  rc = need_b200(&di);
  if (rc != SMB_OK) return rc;
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.q_ts = p->q_strides[0];
  a.q_hs = p->q_strides[1];
  a.k_ts = p->k_strides[0];
  a.k_hs = p->k_strides[1];
  a.v_ts = p->v_strides[0];
  a.v_hs = p->v_strides[1];
  a.slots = reinterpret_cast<const long long*>(p->slots);
  a.positions = reinterpret_cast<const long long*>(p->positions);
  a.inv_freq = p->inv_freq;
  a.rot = rot;
  a.interleaved = p->interleaved;
  a.rope_scale = p->rope_scale;
  a.eps = p->eps;
  a.q_norm = p->q_norm;
  a.k_norm = p->k_norm;
  a.q_out = p->q_out;
  a.status = p->status;
  a.N = N;
  a.Hq = Hq;
  return done(launch_kv_append(a, D, p->dtype == SMB_DTYPE_BF16, p->cache.bits == 4, di.sms,
                               reinterpret_cast<cudaStream_t>(stream), pdl_enabled()));
}

int smb_kv4_read(const smb_paged_cache_t* cache, int dtype, const int64_t* slots, int M, void* out,
                 smb_stream_t stream) {
  if (cache == nullptr) return SMB_ERR_NULL;
  smb_paged_cache_t c = *cache;
  c.v = c.k;
  if (c.bits != 4) return SMB_ERR_DTYPE;
  PagedCacheArgs ca;
  int rc = cache_args(&c, &ca);
  if (rc != SMB_OK) return rc;
  if (!storage(dtype)) return SMB_ERR_DTYPE;
  if (M < 0) return SMB_ERR_SHAPE;
  if (M == 0) return SMB_OK;
  if (slots == nullptr || out == nullptr) return SMB_ERR_NULL;
  if (!aligned16(out)) return SMB_ERR_ALIGN;
  DeviceInfo di;
  rc = need_b200(&di);
  if (rc != SMB_OK) return rc;
  Kv4ReadArgs a{};
  a.cache = ca.k;
  a.num_pages = ca.num_pages;
  a.page_stride = ca.page_stride;
  a.head_stride = ca.head_stride;
  a.token_stride = ca.token_stride;
  a.page_shift = ca.page_shift;
  a.Hkv = ca.Hkv;
  a.slots = reinterpret_cast<const long long*>(slots);
  a.M = M;
  a.out = out;
  return done(launch_kv4_read(a, c.head_dim, dtype == SMB_DTYPE_BF16, reinterpret_cast<cudaStream_t>(stream), pdl_enabled()));
}

size_t smb_paged_attention_workspace_bytes(int N, int B, int Hq, int Hkv, int head_dim, int bits) {
  if (attn_sizes(N, B, Hq, Hkv, head_dim, bits) != SMB_OK) return 0;
  DeviceInfo di;
  if (device_info(&di) != SMB_OK) return 0;
  if (N == 0 || B == 0) return 256;
  // what either kernel takes at these sizes (which one runs depends on the cache's pages too)
  const int g = Hq / Hkv;
  size_t n = attn_ws(plan_attn_mma(N, B, g, head_dim, bits == 4, di.sms), head_dim);
  AttnPlan p;
  if (plan_attn_tc(N, B, g, head_dim, bits == 4, di.sms, &p)) n = std::max(n, attn_ws(p, head_dim));
  if (bits == 4 && plan_attn_q4(N, B, g, head_dim, di.sms, &p)) n = std::max(n, attn_ws(p, head_dim));
  return n;
}

int smb_paged_attention(const smb_attention_args_t* r, smb_stream_t stream) {
  if (r == nullptr) return SMB_ERR_NULL;
  if (r->struct_bytes != sizeof(*r)) return SMB_ERR_SHAPE;
  AttnArgs a{};
  int rc = cache_args(&r->cache, &a.c);
  if (rc != SMB_OK) return rc;
  if (!storage(r->dtype)) return SMB_ERR_DTYPE;
  const int D = r->cache.head_dim, N = r->N, B = r->B;
  rc = attn_sizes(N, B, r->Hq, a.c.Hkv, D, r->cache.bits);
  if (rc != SMB_OK) return rc;
  if (r->max_pages < 0 || r->table_stride < 0) return SMB_ERR_SHAPE;
  // (the kernels count a sequence's keys, and the tile behind its last one, in 32 bits)
  if (r->max_pages > kPagedMaxKeys >> a.c.page_shift) return SMB_ERR_SHAPE;
  if (r->tree != nullptr && (r->tree_words < 1 || r->tree_stride < 0)) return SMB_ERR_SHAPE;
  if (!(r->scale > 0.f) || r->scale > 1e30f) return SMB_ERR_SHAPE;
  if (N == 0 || B == 0) return SMB_OK;
  if (r->q == nullptr || r->out == nullptr || r->kv_lens == nullptr || r->q_starts == nullptr || r->ws == nullptr)
    return SMB_ERR_NULL;
  if (r->max_pages > 0 && r->block_table == nullptr) return SMB_ERR_NULL;
  if (a.c.num_pages == 0) return SMB_ERR_SHAPE;
  if (r->out == r->q) return SMB_ERR_ALIGN;
  if (!aligned16(r->q) || !aligned16(r->out) || !aligned16(r->ws)) return SMB_ERR_ALIGN;
  for (int i = 0; i < 2; ++i)
    if (r->q_strides[i] % 8 != 0 || r->out_strides[i] % 8 != 0) return SMB_ERR_ALIGN;
  DeviceInfo di;
  rc = need_b200(&di);
  if (rc != SMB_OK) return rc;
  a.q = r->q;
  a.q_ts = r->q_strides[0];
  a.q_hs = r->q_strides[1];
  a.N = N;
  a.B = B;
  a.g = r->Hq / a.c.Hkv;
  a.table = r->block_table;
  a.table_stride = r->table_stride;
  a.max_pages = r->max_pages;
  a.kv_lens = r->kv_lens;
  a.q_starts = r->q_starts;
  a.tree = r->tree;
  a.tree_stride = r->tree_stride;
  a.tree_words = r->tree_words;
  a.scale_log2 = r->scale * 1.4426950408889634f;
  a.out = r->out;
  a.o_ts = r->out_strides[0];
  a.o_hs = r->out_strides[1];
  a.lse = r->lse;
  a.status = r->status;
  const bool bits4 = r->cache.bits == 4;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf16 = r->dtype == SMB_DTYPE_BF16;
  AttnPlan p;
  auto use = [&]() {
    a.gs = std::min(a.g, p.rows);
    a.nsub = (a.g + a.gs - 1) / a.gs;
    a.tq = p.rows / a.gs;
    a.part_o = static_cast<float*>(r->ws);
    a.part_ml = a.part_o + static_cast<size_t>(2) * p.grid * p.rows * D;
    a.records = reinterpret_cast<JoinRecord*>(a.part_ml + static_cast<size_t>(4) * p.grid * p.rows);
    a.min_tiles = p.min_tiles;
    a.seg_cost = p.seg_cost;
    return r->ws_bytes >= attn_ws(p, D);
  };
  if (tc_takes(a.c, bits4) && plan_attn_tc(N, B, a.g, D, bits4, di.sms, &p)) {
    if (!use()) return SMB_ERR_WORKSPACE;
    bool fits = false;
    const cudaError_t err = launch_attn_tc(a, p, D, bf16, bits4, st, pdl_enabled(), &fits);
    if (err != cudaSuccess || fits) return done(err);
  }
  if (bits4 && plan_attn_q4(N, B, a.g, D, di.sms, &p)) {
    if (!use()) return SMB_ERR_WORKSPACE;
    return done(launch_attn_q4(a, p, D, bf16, st, pdl_enabled()));
  }
  p = plan_attn_mma(N, B, a.g, D, bits4, di.sms);
  if (!use()) return SMB_ERR_WORKSPACE;
  return done(launch_attn_mma(a, p, D, bf16, bits4, st, pdl_enabled()));
}

}  // extern "C"
