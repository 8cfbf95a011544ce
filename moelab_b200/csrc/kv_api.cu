// C entry points of the 4-bit KV cache (declared in include/moelab_b200.h): argument checks and launches. Nothing is
// allocated and nothing waits for the device, moeb_kv_read_error apart.
#include <math.h>
#include <stdio.h>

#include <algorithm>
#include <atomic>

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

constexpr int DEVICES = 64;  // whose answers are kept

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

int sms() {
    static std::atomic<int> cache[DEVICES];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return 148;
    }
    if (dev < DEVICES && (n = cache[dev].load())) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    if (dev < DEVICES) cache[dev] = n;
    return n;
}

// Resident CTAs per SM of a kernel on the current device, 0 if it cannot run; its dynamic shared memory is allowed on the first
// call. `cache`: the kernel's own.
int resident(std::atomic<int> (&cache)[DEVICES], const void *kern, int threads, size_t smem) {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) {
        if (dev < DEVICES && (n = cache[dev].load())) return n;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess &&
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem) == cudaSuccess && n > 0) {
            if (dev < DEVICES) cache[dev] = n;
            return n;
        }
    }
    cudaGetLastError();
    return 0;
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

int check_seqs(const KvCache &c, int T, const int *cu, const int *lens, bool need_lens, const int *table, long table_row, int B, int P,
               KvSeqs *o) {
    const int o_pshift = c.pshift, kv_heads = c.Hkv;
    if (T < 0 || B < 0 || P < 0) return bad("negative number of rows, sequences or table entries");
    if (T > (1 << 26)) return bad("at most 2^26 rows a call");
    if (T > 0 && B > 0 && ((P > 0 && !table) || (need_lens && !lens))) return bad("table or lens is null");
    if ((long)P << o_pshift > 1L << 30) return bad("at most 2^30 tokens a sequence");
    if ((long)B * kv_heads > 1L << 24) return bad("at most 2^24 pairs of a sequence and a KV head a call");
    if ((((long)P << o_pshift) / 128 + 4) * B > 0x7fffffffL) return bad("the page tables name more than 2^38 tokens");
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

// The kernels that write and read rows: a CTA takes 16 (int4) or 32 (MXFP4) tokens of one head at a time, 4 times where that
// still gives every SM eight CTAs.
int word_heads(const moeb_kv_cache *c) { return KV_BOTH(c->head_dim) ? c->kv_heads : 2 * c->kv_heads; }
int word_passes(const moeb_kv_cache *c, int T) {
    const long rows = c->format == MOEB_KV_Q4 ? 16 : 32, ctas = (T + rows - 1) / rows * word_heads(c);
    return ctas >= 32L * sms() ? 4 : 1;
}
dim3 word_grid(const moeb_kv_cache *c, int T, int passes) {
    const int tokens = (c->format == MOEB_KV_Q4 ? 16 : 32) * passes;
    return dim3((unsigned)((T + tokens - 1) / tokens), (unsigned)word_heads(c));
}

// What a call of moeb_kv_attention launches, from what the host knows: the rows, the page tables' width and the window.
struct Plan {
    long keys;          // keys that one row tile or one sequence's few rows can see, at most
    int few, only;      // sequences of at most `few` (row, head) columns go to the kernel for few rows; all of them do
    int nc, direct;     // its columns per tile; CTAs that share a (sequence, head) (0: all blocks are dealt to all CTAs)
    size_t part, few_bytes;
    long tiles, splits; // row tiles of the kernel for many rows; parts that each one's keys are cut into
    size_t split_bytes;
};
constexpr int FEW_RESIDENT = 4;  // CTAs per SM at most: the workspace has room for their partial results

Plan plan_of(int T, int B, int P, int page_size, int H, int Hkv, int D, int max_q, int window, int sinks, bool cu) {
    Plan p = {};
    const int Gq = H / Hkv;
    const long cols = (long)max_q * Gq, all = (long)P * page_size;
    // The window's keys may start and end inside a block of 128; so may the first tokens'.
    auto seen = [&](long rows) { return window ? std::min(all, (long)window + rows + std::min<long>(sinks, all) + 128 + (sinks ? 128 : 0)) : all; };
    // Sequences whose (row, head) columns fit one or two tensor-core tiles go to the kernel for few rows. Without cu all
    // sequences have T / B rows; with it, and more than one sequence, both kinds may be in the call: over up to 1024 keys
    // the kernel for many rows takes them all (at most 9 key tiles each, against up to two more launches). Single tokens beside
    // one piece of 256 rows, 32 heads on 8, D = 128, this against both kernels: 4 in windows of 128 24 / 34 us, 16 36 / 37, 16 over
    // 1000 keys 59 / 56. It pays while the tiles are about one round of CTAs and loses beyond: 96 over 1000 keys 194 / 125, 96 in
    // windows of 128 with 64 heads on 8, D = 64, 86 / 42.
    p.only = cols <= 16;
    // With more than 16 query heads per KV head no row fits them: one launch, no workspace for the other kernel.
    p.few = p.only ? (int)cols : cu && B > 1 && Gq <= 16 && seen(max_q) > 1024 ? 16 : 0;
    if (p.few) {
        p.nc = cols <= 8 ? 8 : 16;
        // Up to 4 blocks of 128 keys one after the other cost as much as a second launch to join parts of them: one CTA has
        // them, or, where that many CTAs fit the GPU at once, one of a cluster of 8 has (keys to 4096).
        const long keys = seen(std::min(max_q, 16));
        p.direct = keys > 128 && keys <= 4096 && (long)B * Hkv * 8 <= 2L * sms() ? 8 : keys <= 512 ? 1 : 0;
        if (!p.direct) {  // blocks before each sequence, then two partial results per CTA
            p.part = up256(4 * ((size_t)B + 1));
            p.few_bytes = up256(p.part + (size_t)FEW_RESIDENT * sms() * 2 * p.nc * (D + 2) * 4);
        }
    }
    if (!p.only) {
        // Row tiles: with cu each sequence may have one that is not full.
        p.tiles = cu ? (long)T * Gq / KV_PROMPT_ROWS + B : (long)B * (((long)(T / B) * Gq + KV_PROMPT_ROWS - 1) / KV_PROMPT_ROWS);
        const long ctas = p.tiles * Hkv, key_tiles = (seen(KV_PROMPT_ROWS) + 127) / 128;
        // One CTA per SM: where the row tiles alone are less than three waves, their keys are cut into as many parts (8 key tiles
        // or more each) as make the last wave fullest. A key tile takes 2.2 us with heads of 64 and 3.2 us with 128; a part's sums
        // are written and read once more.
        p.splits = 1;
        if (ctas < 3L * sms()) {
            double best = 0;
            const long most = std::max(1L, std::min(key_tiles / 8, ctas * 2 <= sms() ? sms() / std::max(ctas, 1L) : 8L));
            for (long n = 1; n <= most; ++n) {
                const double waves = (double)((ctas * n + sms() - 1) / sms());
                const double us = waves * ((double)key_tiles / n * (D == 64 ? 2.2 : 3.2) + 6.0) + (n > 1 ? 3.0 + (double)n * T * H * D * 8 / 5e6 : 0.0);
                if (n == 1 || us < best * 0.97) {
                    best = us;
                    p.splits = n;
                }
            }
        }
        if (p.splits > 1) p.split_bytes = (size_t)p.splits * T * H * (D + 2) * 4;
    }
    return p;
}

template <int FMT, int D, int NT>
int launch_few(const KvAttnArgs &a, const Plan &p, void *ws, cudaStream_t st) {
    const size_t smem = kv_few_smem<FMT, D, NT>();
    static std::atomic<int> cache[DEVICES];
    const int per = std::min(resident(cache, (const void *)k_kv_attn_few<FMT, D, NT>, 128, smem), FEW_RESIDENT);
    if (!per) return launched(cudaErrorInvalidConfiguration, "kv_attention");
    int *pre = (int *)ws;
    float *part = (float *)((char *)ws + p.part);
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

template <int FMT, int D>
int launch_prompt(const KvAttnArgs &a, const Plan &p, void *ws, cudaStream_t st) {
    const size_t smem = kv_prompt_smem(D);
    static std::atomic<int> cache[DEVICES];
    if (!resident(cache, (const void *)k_kv_attn_prompt<FMT, D>, KV_PROMPT_THREADS, smem))
        return launched(cudaErrorInvalidConfiguration, "kv_attention");
    float *part = p.splits > 1 ? (float *)ws : nullptr;
    cudaError_t e = launch(k_kv_attn_prompt<FMT, D>, dim3((unsigned)(p.tiles * a.c.Hkv), (unsigned)p.splits), KV_PROMPT_THREADS, smem, st, a,
                           (int)p.tiles, part);
    if (e == cudaSuccess && part)
        e = launch(k_kv_attn_join_splits<D>, dim3((unsigned)(((size_t)a.s.T * a.H + 3) / 4)), 128, 0, st, a, (const float *)part, (int)p.splits);
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
    if ((rc = check_seqs(a.c, T, cu, lens, true, table, table_row, B, P, &a.s))) return rc;
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
    if ((rc = check_seqs(a.c, T, cu, nullptr, false, table, table_row, B, P, &a.s))) return rc;
    if (T == 0 || B == 0) return MOEB_OK;
    if (!k || !v || !aligned16(k) || !aligned16(v)) return bad("k and v must be 16-byte aligned");
    a.first = first;
    a.k = (uint16_t *)k;
    a.v = (uint16_t *)v;
    a.passes = word_passes(cache, T);
    return launched(launch(KV_PICK(k_kv_read, cache), word_grid(cache, T, a.passes), 128, 0, stream, a), "kv_read");
}

size_t moeb_kv_attention_workspace_bytes(int T, int B, int P, int page_size, int H, int kv_heads, int head_dim, int max_q,
                                         int window, int sinks, int with_cu) {
    if (T <= 0 || B <= 0 || P < 0 || page_size <= 0 || kv_heads <= 0 || H < kv_heads || head_dim <= 0 || max_q <= 0) return 0;
    const Plan p = plan_of(T, B, P, page_size, H, kv_heads, head_dim, max_q, window, sinks, with_cu != 0);
    return p.few_bytes + p.split_bytes;
}

int moeb_kv_attention(const moeb_kv_cache *cache, const void *q, long q_row, long q_head, int T, int H, const int *cu,
                      const int *lens, const int *table, long table_row, int B, int P, int max_q, float scale, int window,
                      int sinks, const float *sink_logits, void *y, float *lse, void *ws, size_t ws_bytes,
                      cudaStream_t stream) {
    KvAttnArgs a;
    int rc = check_cache(cache, &a.c);
    if (rc) return rc;
    if ((rc = check_seqs(a.c, T, cu, lens, true, table, table_row, B, P, &a.s))) return rc;
    if (H <= 0 || H % cache->kv_heads) return bad("the query heads must be a positive multiple of the cache's kv_heads");
    if (H > 4096) return bad("at most 4096 query heads");
    if ((long)T * H > 0x7fffffffL) return bad("at most 2^31 - 1 rows times query heads a call");
    if (window < 0 || sinks < 0) return bad("window and sinks must not be negative");
    if (!isfinite(scale * 1.4426950408889634f)) return bad("scale must be finite, and below 2^127");
    // what the page tables cannot hold is beyond any window and any first tokens
    const int all = P << a.c.pshift;
    if (window > all) window = 0;
    if (sinks > all) sinks = all;
    if (T == 0 || B == 0) return MOEB_OK;
    if (max_q <= 0) return bad("max_q must be positive");
    if (!rows_ok(q, q_row, q_head))
        return bad("q must be 16-byte aligned, with row and head strides that are multiples of 8 elements");
    if (!y || !aligned16(y)) return bad("y must be 16-byte aligned");
    const Plan p = plan_of(T, B, P, cache->page_size, H, cache->kv_heads, cache->head_dim, max_q, window, sinks, cu != nullptr);
    if (p.few_bytes + p.split_bytes > 0 && (!ws || !aligned16(ws))) return bad("the workspace must be 16-byte aligned");
    if (ws_bytes < p.few_bytes + p.split_bytes)
        return bad("the workspace is too small: see moeb_kv_attention_workspace_bytes");
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
    a.few = p.few;
    a.only = p.only;
    a.direct = p.direct;
    const bool q4 = cache->format == MOEB_KV_Q4, d64 = cache->head_dim == 64;
    if (p.few) {
        if (p.nc == 8)
            rc = q4 ? (d64 ? launch_few<FMT_Q4, 64, 1>(a, p, ws, stream) : launch_few<FMT_Q4, 128, 1>(a, p, ws, stream))
                    : (d64 ? launch_few<FMT_FP4, 64, 1>(a, p, ws, stream) : launch_few<FMT_FP4, 128, 1>(a, p, ws, stream));
        else
            rc = q4 ? (d64 ? launch_few<FMT_Q4, 64, 2>(a, p, ws, stream) : launch_few<FMT_Q4, 128, 2>(a, p, ws, stream))
                    : (d64 ? launch_few<FMT_FP4, 64, 2>(a, p, ws, stream) : launch_few<FMT_FP4, 128, 2>(a, p, ws, stream));
        if (rc || p.only) return rc;
    }
    void *rest = (char *)ws + p.few_bytes;
    return q4 ? (d64 ? launch_prompt<FMT_Q4, 64>(a, p, rest, stream) : launch_prompt<FMT_Q4, 128>(a, p, rest, stream))
              : (d64 ? launch_prompt<FMT_FP4, 64>(a, p, rest, stream) : launch_prompt<FMT_FP4, 128>(a, p, rest, stream));
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
