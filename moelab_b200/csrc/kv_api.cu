// C entry points of the 4-bit KV cache (declared in include/moelab_b200.h): argument checks and launches. Nothing is
// allocated and nothing waits for the device, moeb_kv_read_error apart.
#include <math.h>
#include <stdio.h>

#include <algorithm>
#include <map>
#include <mutex>

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
template <typename... K, typename... A>
cudaError_t launch_cluster(void (*kern)(K...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}
template <typename... K, typename... A>
cudaError_t launch(void (*kern)(K...), dim3 grid, int threads, size_t smem, cudaStream_t st, const A &...args) {
    return launch_cluster(kern, grid, threads, smem, 1, st, args...);
}

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

int sms() {
    static std::mutex mu;
    static std::map<int, int> cache;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return 148;
    }
    std::lock_guard<std::mutex> lk(mu);
    int &n = cache[dev];
    if (!n && (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)) n = 148;
    return n;
}

// Resident CTAs per SM of a kernel on the current device; its dynamic shared memory is allowed on the first call.
int resident(const void *kern, int threads, size_t smem) {
    static std::mutex mu;
    static std::map<std::pair<const void *, int>, int> cache;
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> lk(mu);
    int &n = cache[{kern, dev}];
    if (!n) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem) != cudaSuccess || n < 1)
            n = 0;
    }
    return n;
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

// The kernels that write and read rows: a CTA takes 16 (int4) or 32 (MXFP4) tokens of one head's K or V at a time, 4 times
// where that still gives every SM eight CTAs.
int word_passes(const moeb_kv_cache *c, int T) {
    const long ctas = (((long)T + (c->format == MOEB_KV_Q4 ? 15 : 31)) / (c->format == MOEB_KV_Q4 ? 16 : 32)) * 2 * c->kv_heads;
    return ctas >= 32L * sms() ? 4 : 1;
}
dim3 word_grid(const moeb_kv_cache *c, int T, int passes) {
    const int tokens = (c->format == MOEB_KV_Q4 ? 16 : 32) * passes;
    return dim3((unsigned)((T + tokens - 1) / tokens), 2u * c->kv_heads);
}

// Workspace of the kernel for few rows: blocks before each sequence, then two partial results per CTA.
struct FewLayout {
    size_t part, total;
};
constexpr int FEW_RESIDENT = 3;  // CTAs per SM at most (the kernel's launch bound)
FewLayout few_layout(int B, int nc, int D) {
    FewLayout l;
    l.part = up256(4 * ((size_t)B + 1));
    l.total = l.part + (size_t)FEW_RESIDENT * sms() * 2 * nc * (D + 2) * 4;
    return l;
}

template <int FMT, int D, int NT>
int launch_few(const KvAttnArgs &a, void *ws, cudaStream_t st) {
    const size_t smem = kv_few_smem<FMT, D, NT>();
    const int per = resident((const void *)k_kv_attn_few<FMT, D, NT>, 128, smem);
    if (!per) return launched(cudaErrorInvalidConfiguration, "kv_attention");
    const FewLayout l = few_layout(a.s.B, 8 * NT, D);
    int *pre = (int *)ws;
    float *part = (float *)((char *)ws + l.part);
    // at most one block of 128 keys per CTA: the page tables' width bounds the blocks, each (sequence, head) has 2 more in the count
    const long most = (long)a.s.B * a.c.Hkv * ((((long)a.s.P << a.c.pshift) >> 7) + 4);
    const int grid = (int)(most < (long)per * sms() ? most : (long)per * sms());
    if (a.direct)
        return launched(launch_cluster(k_kv_attn_few<FMT, D, NT>, dim3(a.s.B * a.c.Hkv * a.direct), 128, smem, a.direct, st, a, pre, part),
                        "kv_attention");
    cudaError_t e = launch(k_kv_attn_few<FMT, D, NT>, dim3(grid), 128, smem, st, a, pre, part);
    if (e == cudaSuccess)
        e = launch(k_kv_attn_join<D, NT>, dim3(a.s.B * a.c.Hkv, a.few), 256, 0, st, a, (const int *)pre, (const float *)part, grid);
    return launched(e, "kv_attention");
}

// Row tiles of the kernel for many rows, and into how many parts each tile's keys are cut: as many as give every SM a
// CTA, where the rows alone do not.
long prompt_tiles(int T, int B, int Gq, bool cu) {
    return cu ? (long)T * Gq / KV_PROMPT_ROWS + B : (long)B * (((long)(T / B) * Gq + KV_PROMPT_ROWS - 1) / KV_PROMPT_ROWS);
}
long prompt_splits(long tiles, int Hkv) { return tiles * Hkv * 2 > sms() ? 1 : sms() / (tiles * Hkv); }

template <int FMT, int D>
int launch_prompt(const KvAttnArgs &a, void *ws, cudaStream_t st) {
    const size_t smem = kv_prompt_smem(D);
    if (!resident((const void *)k_kv_attn_prompt<FMT, D>, KV_PROMPT_THREADS, smem))
        return launched(cudaErrorInvalidConfiguration, "kv_attention");
    const long tiles = prompt_tiles(a.s.T, a.s.B, a.Gq, a.s.cu != nullptr);
    const long keys = (((long)a.s.P << a.c.pshift) + 127) >> 7;  // key tiles at most
    long ns = prompt_splits(tiles, a.c.Hkv);
    if (ns > keys) ns = keys < 1 ? 1 : keys;
    float *part = ns > 1 ? (float *)ws : nullptr;
    cudaError_t e = launch(k_kv_attn_prompt<FMT, D>, dim3((unsigned)(tiles * a.c.Hkv), (unsigned)ns), KV_PROMPT_THREADS, smem, st, a,
                           (int)tiles, part);
    if (e == cudaSuccess && ns > 1)
        e = launch(k_kv_attn_join_splits<D>, dim3((unsigned)(((size_t)a.s.T * a.H + 3) / 4)), 128, 0, st, a, (const float *)part, (int)ns);
    return launched(e, "kv_attention");
}

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
    a.passes = word_passes(cache, T);
    return launched(launch(KV_PICK(k_kv_write, cache), word_grid(cache, T, a.passes), 128, 0, stream, a), "kv_write");
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
    a.passes = word_passes(cache, T);
    return launched(launch(KV_PICK(k_kv_read, cache), word_grid(cache, T, a.passes), 128, 0, stream, a), "kv_read");
}

size_t moeb_kv_attention_workspace_bytes(int T, int B, int H, int kv_heads, int head_dim, int max_q) {
    if (T <= 0 || B <= 0 || H <= 0 || kv_heads <= 0 || head_dim <= 0 || max_q <= 0) return 0;
    const int Gq = H / kv_heads;
    const long cols = (long)max_q * Gq;
    size_t n = up256(few_layout(B, cols <= 8 ? 8 : 16, head_dim).total);
    if (cols > 16) {
        const long tiles = T % B ? prompt_tiles(T, B, Gq, true) : std::min(prompt_tiles(T, B, Gq, true), prompt_tiles(T, B, Gq, false));
        const long ns = prompt_splits(tiles, kv_heads);
        if (ns > 1) n += (size_t)ns * T * H * (head_dim + 2) * 4;
    }
    return n;
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
    if (!ws || !aligned16(ws)) return bad("the workspace must be 16-byte aligned");
    a.q = (const uint16_t *)q;
    a.q_row = q_row;
    a.q_head = q_head;
    a.H = H;
    a.Gq = H / cache->kv_heads;
    a.Gdiv = a.Gq == 1 ? 0u : (unsigned)((0x100000000ull + a.Gq - 1) / a.Gq);
    a.scale = scale * 1.4426950408889634f;
    a.window = window;
    a.sinks = sinks;
    a.sink_logits = sink_logits;
    a.y = (uint16_t *)y;
    a.lse = lse;
    // Sequences whose (row, head) columns fit one or two tensor-core tiles go to the kernel for few rows. Without cu all
    // sequences have T / B rows; with it, and more than one sequence, both kinds may be in the call.
    const long cols = (long)max_q * a.Gq;
    const bool only_few = cols <= 16, both = !only_few && cu && B > 1;
    a.few = only_few ? (int)cols : both ? 16 : 0;
    if (a.few) {
        const bool one = cols <= 8;
        a.only = only_few;
        // Up to 4 blocks of 128 keys one after the other cost as much as a second launch to join parts of them: one CTA has
        // them, or, where that many CTAs fit the GPU at once, one of a cluster of 8 has (keys to 4096). The bound is known here from
        // the page tables' width, or from the window (its keys may start and end inside a block).
        long keys = (long)P << a.c.pshift;
        if (window) {
            const long seen = (long)window + std::min<long>(max_q, 16) + std::min<long>(sinks, keys);
            keys = std::min(keys, seen + 128 + (sinks ? 128 : 0));
        }
        const long heads = (long)B * a.c.Hkv;
        a.direct = keys > 128 && keys <= 4096 && heads * 8 <= 2L * sms() ? 8 : keys <= 512 ? 1 : 0;
        rc = cache->format == MOEB_KV_Q4
                 ? (cache->head_dim == 64 ? (one ? launch_few<FMT_Q4, 64, 1>(a, ws, stream) : launch_few<FMT_Q4, 64, 2>(a, ws, stream))
                                          : (one ? launch_few<FMT_Q4, 128, 1>(a, ws, stream) : launch_few<FMT_Q4, 128, 2>(a, ws, stream)))
                 : (cache->head_dim == 64 ? (one ? launch_few<FMT_FP4, 64, 1>(a, ws, stream) : launch_few<FMT_FP4, 64, 2>(a, ws, stream))
                                          : (one ? launch_few<FMT_FP4, 128, 1>(a, ws, stream) : launch_few<FMT_FP4, 128, 2>(a, ws, stream)));
        if (rc) return rc;
    }
    if (only_few) return MOEB_OK;
    void *rest = (char *)ws + up256(few_layout(B, 16, cache->head_dim).total);
    return cache->format == MOEB_KV_Q4
               ? (cache->head_dim == 64 ? launch_prompt<FMT_Q4, 64>(a, rest, stream) : launch_prompt<FMT_Q4, 128>(a, rest, stream))
               : (cache->head_dim == 64 ? launch_prompt<FMT_FP4, 64>(a, rest, stream) : launch_prompt<FMT_FP4, 128>(a, rest, stream));
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
