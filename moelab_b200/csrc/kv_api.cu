// C entry points of the 4-bit KV cache (declared in include/moelab_b200.h): argument checks and launches. Nothing is
// allocated and nothing waits for the device, moeb_kv_read_error apart.
#include <math.h>
#include <stdio.h>

#include "../../include/moelab_b200.h"
#include "kv.cuh"

using namespace moeb;

namespace {

int bad(const char *msg, int code = MOEB_EINVAL) {
    set_error(msg);
    return code;
}

int launched(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return MOEB_OK;
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", what, cudaGetErrorString(e));
    cudaGetLastError();
    set_error(msg);
    return MOEB_ELAUNCH;
}

// Programmatic dependent launch, as every kernel of this library: the kernel waits (pdl_wait) before it reads or
// writes anything.
template <typename A>
cudaError_t launch(void (*kern)(A), dim3 grid, int threads, size_t smem, cudaStream_t st, const A &args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args);
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int check_cache(const moeb_kv_cache *c, KvCache *o) {
    if (!c) return bad("the cache is null");
    if (!c->kq || !c->ks || !c->vq || !c->vs || !c->err) return bad("a cache array is null");
    if (!aligned16(c->kq) || !aligned16(c->ks) || !aligned16(c->vq) || !aligned16(c->vs))
        return bad("cache arrays must be 16-byte aligned");
    if (c->format != MOEB_KV_Q4 && c->format != MOEB_KV_MXFP4) return bad("unknown cache format", MOEB_EUNSUP);
    if (c->head_dim != 64 && c->head_dim != 128) return bad("head_dim must be 64 or 128", MOEB_EUNSUP);
    if (c->page_size < 16 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
        return bad("page_size must be a power of two from 16 to 4096");
    if (c->pages <= 0 || c->kv_heads <= 0 || c->kv_heads > 1024) return bad("pages and kv_heads must be positive, kv_heads at most 1024");
    o->kq = (uint32_t *)c->kq;
    o->vq = (uint32_t *)c->vq;
    o->ks = c->ks;
    o->vs = c->vs;
    o->err = c->err;
    o->pages = c->pages;
    o->pshift = __builtin_ctz((unsigned)c->page_size);
    o->Hkv = c->kv_heads;
    return MOEB_OK;
}

int check_seqs(int T, const int *cu, const int *lens, bool need_lens, const int *table, long table_row, int B, int P, KvSeqs *o) {
    if (T < 0 || B < 0 || P < 0) return bad("negative number of rows, sequences or table entries");
    if (T > (1 << 26)) return bad("at most 2^26 rows a call");
    if (T > 0 && B > 0 && (!table || (need_lens && !lens))) return bad("table or lens is null");
    if (B > 1 && table_row < P) return bad("table rows overlap");
    if (!cu && B > 0 && T % B) return bad("without cu every sequence has the same number of rows: T must be a multiple of B");
    o->cu = cu;
    o->lens = lens;
    o->table = table;
    o->trow = table_row;
    o->B = B;
    o->P = P;
    o->T = T;
    o->each = !cu && B > 0 ? T / B : 0;
    return MOEB_OK;
}

#define KV_PICK(kern, c) \
    ((c)->format == MOEB_KV_Q4 ? ((c)->head_dim == 64 ? kern<FMT_Q4, 64> : kern<FMT_Q4, 128>) \
                               : ((c)->head_dim == 64 ? kern<FMT_FP4, 64> : kern<FMT_FP4, 128>))

bool rows_ok(const void *p, long row, long head) { return p && aligned16(p) && row % 8 == 0 && head % 8 == 0; }

}  // namespace

extern "C" {

int moeb_kv_write(const moeb_kv_cache *cache, const void *k, long k_row, long k_head, const void *v, long v_row,
                  long v_head, int T, const int *cu, const int *lens, const int *table, long table_row, int B, int P,
                  cudaStream_t stream) {
    KvWriteArgs a;
    int rc = check_cache(cache, &a.c);
    if (rc) return rc;
    if ((rc = check_seqs(T, cu, lens, true, table, table_row, B, P, &a.s))) return rc;
    if (T == 0 || B == 0) return MOEB_OK;
    if (!rows_ok(k, k_row, k_head) || !rows_ok(v, v_row, v_head))
        return bad("k and v must be 16-byte aligned, with row and head strides that are multiples of 8 elements");
    a.k = (const uint16_t *)k;
    a.v = (const uint16_t *)v;
    a.k_row = k_row;
    a.k_head = k_head;
    a.v_row = v_row;
    a.v_head = v_head;
    const long n = (long)T * 2 * cache->kv_heads * (cache->head_dim / 8);
    return launched(launch(KV_PICK(k_kv_write, cache), dim3((unsigned)((n + 127) / 128)), 128, 0, stream, a), "kv_write");
}

int moeb_kv_read(const moeb_kv_cache *cache, int T, const int *cu, const int *first, const int *table, long table_row,
                 int B, int P, void *k, void *v, cudaStream_t stream) {
    KvReadArgs a;
    int rc = check_cache(cache, &a.c);
    if (rc) return rc;
    if ((rc = check_seqs(T, cu, nullptr, false, table, table_row, B, P, &a.s))) return rc;
    if (T == 0 || B == 0) return MOEB_OK;
    if (!k || !v || !aligned16(k) || !aligned16(v)) return bad("k and v must be 16-byte aligned");
    a.first = first;
    a.k = (uint16_t *)k;
    a.v = (uint16_t *)v;
    const long n = (long)T * 2 * cache->kv_heads * (cache->head_dim / 8);
    return launched(launch(KV_PICK(k_kv_read, cache), dim3((unsigned)((n + 127) / 128)), 128, 0, stream, a), "kv_read");
}

size_t moeb_kv_attention_workspace_bytes(int T, int B, int H, int kv_heads, int head_dim, int max_q) {
    (void)T; (void)B; (void)H; (void)kv_heads; (void)head_dim; (void)max_q;
    return 0;
}

int moeb_kv_attention(const moeb_kv_cache *cache, const void *q, long q_row, long q_head, int T, int H, const int *cu,
                      const int *lens, const int *table, long table_row, int B, int P, int max_q, float scale, int window,
                      int sinks, const float *sink_logits, void *y, float *lse, void *ws, size_t ws_bytes,
                      cudaStream_t stream) {
    KvAttnArgs a;
    int rc = check_cache(cache, &a.c);
    if (rc) return rc;
    if ((rc = check_seqs(T, cu, lens, true, table, table_row, B, P, &a.s))) return rc;
    if (H <= 0 || H % cache->kv_heads) return bad("the query heads must be a positive multiple of the cache's kv_heads");
    if (H > 4096) return bad("at most 4096 query heads");
    if (window < 0 || sinks < 0) return bad("window and sinks must not be negative");
    if (!isfinite(scale)) return bad("scale must be finite");
    if (T == 0 || B == 0) return MOEB_OK;
    if (max_q <= 0) return bad("max_q must be positive");
    if (!rows_ok(q, q_row, q_head))
        return bad("q must be 16-byte aligned, with row and head strides that are multiples of 8 elements");
    if (!y || !aligned16(y)) return bad("y must be 16-byte aligned");
    if (ws_bytes < moeb_kv_attention_workspace_bytes(T, B, H, cache->kv_heads, cache->head_dim, max_q))
        return bad("the workspace is too small: see moeb_kv_attention_workspace_bytes");
    (void)ws;
    a.q = (const uint16_t *)q;
    a.q_row = q_row;
    a.q_head = q_head;
    a.H = H;
    a.Gq = H / cache->kv_heads;
    a.scale = scale * 1.4426950408889634f;
    a.window = window;
    a.sinks = sinks;
    a.sink_logits = sink_logits;
    a.y = (uint16_t *)y;
    a.lse = lse;
    return launched(launch(KV_PICK(k_kv_attn_rows, cache), dim3(T, H), 128, 0, stream, a), "kv_attention");
}

int moeb_kv_read_error(const moeb_kv_cache *cache, unsigned *out, cudaStream_t stream) {
    KvCache c;
    const int rc = check_cache(cache, &c);
    if (rc) return rc;
    if (!out) return bad("out is null");
    cudaError_t e = cudaMemcpyAsync(out, c.err, sizeof(unsigned), cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(c.err, 0, sizeof(unsigned), stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    return launched(e, "kv_read_error");
}

}  // extern "C"
