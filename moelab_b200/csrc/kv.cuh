// The 4-bit KV cache: its layout, the lookups every cache kernel shares, and the kernels' argument blocks.
//
// A cache holds pages of `page` tokens (a power of two, at least 16) of one layer, and K and V apart. A row is one
// (token, KV head): D = 64 or 128 values in W = D / 8 code words plus its group parameters,
//   codes  uint32 [pages][Hkv][page][W]
//   int4 parameters   uint32 [pages][Hkv][page][D / 64]  (bf16 scale | bf16 bias << 16; value = scale * code + bias)
//   MXFP4 parameters  uint8  [pages][Hkv][page][D / 32]  (E8M0; value = E2M1(code) * 2^(byte - 127))
// so a page's tokens of one head are one contiguous block, and 16 tokens (a tensor-core tile's rows) are D * 8 bytes in a
// row. The order inside a row is the one the decode kernel's registers want (kv_attn.cu):
//   int4: words of 8 values, element 2 p at nibble p, element 2 p + 1 at nibble p + 4 (as in the expert weights); word w = 0 .. 7
//     of group g (of G = D / 64) at w * G + g
//   MXFP4: half-words of 4 values, element i at nibble i; half-word u = 0 .. 7 of group g (of H = D / 32) at half-word u * H + g
// With it a lane's codes of one key (1 / 4 of the row for K, 1 / 8 for V) are one load of 4 to 16 bytes, and hold the same part
// of every group.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace moeb {

enum : uint32_t {
    ERR_PAGE = 4u,  // a token's page is outside the table or the cache
    ERR_ROWS = 8u,  // a sequence has more rows than the call's max_q: they were passed over
};

struct KvCache {
    uint32_t *kq, *vq;
    void *ks, *vs;
    unsigned *err;
    int pages, pshift, Hkv;  // page = 1 << pshift tokens
};
// Rows of a call: sequence b has rows cu[b] .. cu[b + 1] - 1 (cu == null: `each` rows per sequence), its page ids are
// table[b * trow ..], P of them.
struct KvSeqs {
    const int *cu, *lens, *table;
    long trow;
    int B, P, T, each;
};

// pairs of fp32 in one 64-bit register: one instruction for two sums or products
MOEB_DEV uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
MOEB_DEV void unpair(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
MOEB_DEV uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
MOEB_DEV uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
MOEB_DEV uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

MOEB_DEV int kv_clamp_row(int v, int T) { return v < 0 ? 0 : (v > T ? T : v); }
// rows [r0, r1) of sequence b, inside [0, T)
MOEB_DEV void kv_rows(const KvSeqs &s, int b, int &r0, int &r1) {
    if (s.cu) {
        r0 = kv_clamp_row(s.cu[b], s.T);
        r1 = kv_clamp_row(s.cu[b + 1], s.T);
        if (r1 < r0) r1 = r0;
    } else {
        r0 = b * s.each;
        r1 = r0 + s.each;
    }
}
// sequence of row t, or -1 where it belongs to none; r0 / r1: the sequence's rows
MOEB_DEV int kv_seq_of(const KvSeqs &s, int t, int &r0, int &r1) {
    if (!s.cu) {
        const int b = t / s.each;
        kv_rows(s, b, r0, r1);
        return b;
    }
    // the last b with cu[b] <= t; first where it is when all sequences have as many rows
    const int guess = min((int)__fdividef((float)t * (float)s.B, (float)s.T), s.B - 1);
    if (s.cu[guess] <= t && t < s.cu[guess + 1] && s.cu[guess + 1] <= s.T && s.cu[guess] >= 0) {
        r0 = s.cu[guess];
        r1 = s.cu[guess + 1];
        return guess;
    }
    int lo = 0, hi = s.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s.cu[mid] <= t) lo = mid; else hi = mid;
    }
    kv_rows(s, lo, r0, r1);
    return t >= r0 && t < r1 ? lo : -1;
}
// Row index ((page * Hkv + h) * page_size + offset) of position p of sequence b; -1 where its page is not valid.
MOEB_DEV long kv_page(const KvCache &c, const KvSeqs &s, int b, int p) {
    const int pi = p >> c.pshift;
    if (pi >= s.P) return -1;
    const int id = s.table[(size_t)b * s.trow + pi];
    return id >= 0 && id < c.pages ? (long)id : -1;
}
MOEB_DEV size_t kv_row(const KvCache &c, long page, int h, int p) {
    return (((size_t)page * c.Hkv + h) << c.pshift) + (size_t)(p & ((1 << c.pshift) - 1));
}

// 2^(byte - 127), NaN for 255
MOEB_DEV float kv_e8m0(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
// the 8 values of code word `word` in their natural order. int4: the code into the low bits of 2^23, one exact subtraction and
// one fused product; MXFP4: E2M1 to fp16 (exact) to fp32, times the power of two
template <int FMT>
MOEB_DEV void kv_word_values(uint32_t word, uint32_t par, float (&o)[8]) {
    if (FMT == FMT_Q4) {
        const float s = bf16lo(par), b = bf16hi(par);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t c = (word >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u;
            o[i] = __fmaf_rn(s, __uint_as_float(0x4B000000u | c) - 8388608.f, b);
        }
    } else {
        const float s = kv_e8m0(par);
        uint32_t h[4];
        asm("{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %4;\n cvt.rn.f16x2.e2m1x2 %0, b0;\n cvt.rn.f16x2.e2m1x2 %1, b1;\n"
            " cvt.rn.f16x2.e2m1x2 %2, b2;\n cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
            : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
            : "r"(word));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
            o[2 * i] = f.x * s;
            o[2 * i + 1] = f.y * s;
        }
    }
}
// Rows of 64 values: a thread of the kernels that write and read rows has both K and V of its (token, head), so that there is as
// much work per lookup as with 128.
#define KV_BOTH(D) ((D) == 64)
struct KvWriteArgs {
    KvCache c;
    KvSeqs s;
    const uint16_t *k, *v;
    long k_row, k_head, v_row, v_head;  // strides in elements
    int passes;                         // of a CTA's rows
};
struct KvReadArgs {
    KvCache c;
    KvSeqs s;          // s.lens = null: rows start at first[b] (null: 0)
    const int *first;
    uint16_t *k, *v;   // [T][Hkv][D]
    int passes;
};
struct KvAttnArgs {
    KvCache c;
    KvSeqs s;
    const uint16_t *q;
    long q_row, q_head;
    int H, Gq;         // query heads, query heads per KV head
    unsigned Gdiv;     // ceil(2^32 / Gq), 0 for 1: see kv_div
    float scale;       // of the scores, times log2(e)
    int window, sinks;
    int few;           // sequences of at most this many (row, head) columns are the kernel for few rows', the others not
    int only;          // that kernel has the call to itself (longer sequences are an error)
    int direct;        // CTAs that share a (sequence, head) in its own cluster; 0: all blocks are dealt to all CTAs
    const float *sink_logits;  // [H] or null
    uint16_t *y;       // [T][H][D]
    float *lse;        // [T][H] or null
};
// n / Gq for n < 2^16 (columns and rows of a tile): the product of n and 2^32 / Gq, rounded up, is less than 1 / Gq too large
MOEB_DEV int kv_div(int n, unsigned div) { return div ? (int)__umulhi((unsigned)n, div) : n; }
// Four values of one row's result: v is the sum of weights 2^(score - M) times values, L the sum of the weights.
template <int D>
MOEB_DEV void kv_finish(const KvAttnArgs &a, int t, int head, int d4, float4 v, float M, float L) {
    if (a.sink_logits) {
        const float s = a.sink_logits[head] * 1.4426950408889634f, N = fmaxf(M, s), use = N == -INFINITY ? 0.f : N;
        const float f = exp2f(M - use);
        v.x *= f;
        v.y *= f;
        v.z *= f;
        v.w *= f;
        L = L * f + exp2f(s - use);
        M = N;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;  // a row that sees nothing: zeros
    const size_t row = (size_t)t * a.H + head;
    *reinterpret_cast<uint2 *>(a.y + row * D + 4 * d4) = make_uint2(pack_bf2(v.x * inv, v.y * inv), pack_bf2(v.z * inv, v.w * inv));
    if (a.lse && d4 == 0) a.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}
// first value of the 4 that physical half-word u of a row holds
template <int FMT, int D>
MOEB_DEV int kv_dim(int u) {
    return FMT == FMT_Q4 ? 64 * ((u >> 1) % (D / 64)) + 8 * ((u >> 1) / (D / 64)) + 4 * (u & 1) : 32 * (u % (D / 32)) + 4 * (u / (D / 32));
}
// its values in row `row` of an array
template <int FMT, int D>
MOEB_DEV float4 kv_four(const void *codes, const void *pars, size_t row, int u) {
    // MXFP4: a 32-bit load and a shift; from a 16-bit load nvcc 12.9 made zeros of the conversions' bytes
    const uint32_t word = static_cast<const uint32_t *>(codes)[row * (D / 8) + (u >> 1)] >> ((FMT == FMT_Q4 ? 8 : 16) * (u & 1));
    const uint32_t par = FMT == FMT_Q4 ? static_cast<const uint32_t *>(pars)[row * (D / 64) + (u >> 1) % (D / 64)]
                                       : static_cast<const uint8_t *>(pars)[row * (D / 32) + u % (D / 32)];
    float y[8];
    kv_word_values<FMT>(word, par, y);
    return make_float4(y[0], y[1], y[2], y[3]);
}
// A row's attention in fp32 throughout, by one warp: its keys in blocks [k0, k1) of 128, block k from token 128 k on for k < ns
// and 128 (k + skip) for the others. For keys and values whose sizes are too far apart for the tensor cores' fp16 operands (see
// KV_SPREAD) and for scores of sizes that no softmax has (KV_FAR); ordinary ones never come here, so it is written to be short
// and every key's score is a sum over the lanes. v: values kv_dim(lane) .. + 3 of the sum of weights 2^(score - M) times
// values, L: the sum of the weights, in every lane.
struct KvSum {
    float4 v;
    float M, L;
};
template <int FMT, int D>
MOEB_DEV KvSum kv_exact(const KvAttnArgs &a, int b, int h, const uint16_t *q, int pos, int k0, int k1, int ns, int skip) {
    const int lane = threadIdx.x & 31, u = lane % (D / 4);
    const uint2 w = *reinterpret_cast<const uint2 *>(q + kv_dim<FMT, D>(u));
    float4 x = make_float4(bf16lo(w.x), bf16hi(w.x), bf16lo(w.y), bf16hi(w.y));
    const float top = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    const bool bad = __any_sync(0xffffffffu, !(top < INFINITY) || x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w);
    if (bad) x = make_float4(__uint_as_float(0x7fffffffu), 0.f, 0.f, 0.f);  // NaN, whatever it meets
    if (lane >= D / 4 || (a.scale == 0.f && !bad)) x = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float M = -INFINITY, L = 0.f;
#pragma unroll 1
    for (int k = k0; k < k1; ++k) {
#pragma unroll 1
        for (int j0 = 128 * (k < ns ? k : k + skip), end = min(j0 + 128, pos + 1); j0 < end; j0 += 16) {
            const long page = kv_page(a.c, a.s, b, j0);
            if (page < 0 || (a.window && j0 + 15 <= pos - a.window && j0 >= a.sinks)) continue;
            const size_t row = kv_row(a.c, page, h, j0);
#pragma unroll 1
            for (int i = 0; i < 16; i += 4) {
                float s[4];
                float4 y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 c = kv_four<FMT, D>(a.c.kq, a.c.ks, row + i + e, u);
                    y[e] = kv_four<FMT, D>(a.c.vq, a.c.vs, row + i + e, u);
                    s[e] = fmaf(x.x, c.x, fmaf(x.y, c.y, fmaf(x.z, c.z, x.w * c.w)));
                    if (lane >= D / 4) s[e] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
#pragma unroll
                    for (int o = 16; o; o >>= 1) s[e] += __shfl_xor_sync(0xffffffffu, s[e], o);
                    const int j = j0 + i + e;
                    if (j > pos || (a.window && j <= pos - a.window && j >= a.sinks)) continue;
                    const float t = s[e] * a.scale, N = fmaxf(M, t), use = N == -INFINITY ? 0.f : N, f = exp2f(M - use), p = exp2f(t - use);
                    M = N;
                    L = fmaf(L, f, p);
                    v.x = fmaf(v.x, f, p * y[e].x);
                    v.y = fmaf(v.y, f, p * y[e].y);
                    v.z = fmaf(v.z, f, p * y[e].z);
                    v.w = fmaf(v.w, f, p * y[e].w);
                }
            }
        }
    }
    return {v, M, L};
}
// The tensor cores' fp16 operands hold groups of values up to 2^KV_SPREAD apart: the largest is put near 2^8, one 2^18 smaller is
// near 2^-10 and rounds by 2^-25, 2^-15 of it (fp16's own rounding: 2^-11 of each value). Groups further below the largest, but
// not below 2^-120 (those may count as zeros), make a run of keys uneven: kv_exact has it. The largest may be a key's that the
// row does not see, or hardly looks at, so that what it would round away can be all of the row's result.
constexpr int KV_SPREAD = 18;
// A weight is 2^(score * scale - m) in one fused product, m being a score * scale that was rounded: off by 2^-8 at this size of m
// (in powers of two, as the fp32 score itself), and by whole powers above 2^24, where the largest weight could pass any range.
// kv_exact subtracts what it has rounded.
constexpr float KV_FAR = 65536.f;
constexpr uint32_t KV_ZERO = 7u << 23;  // bits of 2^-120
template <int FMT, int D>
__global__ void k_kv_write(const KvWriteArgs a);
template <int FMT, int D>
__global__ void k_kv_read(const KvReadArgs a);
template <int FMT, int D, int NT>
__global__ void k_kv_attn_few(const KvAttnArgs a, int *pre, float *part);
template <int D, int NT>
__global__ void k_kv_attn_join(const KvAttnArgs a, const int *pre, const float *part, int grid);
template <int FMT, int D, int NT>
size_t kv_few_smem();
template <int FMT, int D>
__global__ void k_kv_attn_prompt(const KvAttnArgs a, int tiles, float *part);
template <int D>
__global__ void k_kv_attn_join_splits(const KvAttnArgs a, const float *part, int ns);
size_t kv_prompt_smem(int D);
constexpr int KV_PROMPT_ROWS = 256, KV_PROMPT_THREADS = 896;

}  // namespace moeb
