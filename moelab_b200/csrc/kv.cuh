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
