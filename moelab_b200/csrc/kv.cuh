// The 4-bit KV cache: its layout, the lookups every cache kernel shares, and the kernels' argument blocks.
//
// A cache holds pages of `page` tokens (a power of two, at least 16) of one layer, and K and V apart. A row is one
// (token, KV head): D = 64 or 128 values in W = D / 8 code words plus its group parameters,
//   codes  uint32 [pages][Hkv][page][W]
//   int4 parameters   uint32 [pages][Hkv][page][D / 64]  (bf16 scale | bf16 bias << 16; value = scale * code + bias)
//   MXFP4 parameters  uint8  [pages][Hkv][page][D / 32]  (E8M0; value = E2M1(code) * 2^(byte - 127))
// so a page's tokens of one head are one contiguous block, and 16 tokens (a tensor-core tile's rows) are D * 8 bytes in a
// row. The order inside a row is the one the decode kernel's registers want (kv_attn.cu):
//   K: word w of group g (64 values) at (w / 2) * 2 * G + 2 * g + w % 2, G = D / 64: a lane's words (2 c, 2 c + 1 of every
//      group) are one 8- or 16-byte load
//   V: word w of group g at w * G + g: a lane's words (w of every group) are one 4- or 8-byte load
//   int4 word: element 2 p at nibble p, element 2 p + 1 at nibble p + 4 (as in the expert weights);
//   MXFP4 word: element i at nibble i (a byte is a pair for the E2M1 -> fp16 conversion)
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace moeb {

enum : uint32_t { ERR_PAGE = 4u };  // a visible token's page is outside the table or the cache

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

__host__ __device__ __forceinline__ int kv_kpos(int w, int G) { return ((w & 7) >> 1) * 2 * G + 2 * (w >> 3) + (w & 1); }
__host__ __device__ __forceinline__ int kv_vpos(int w, int G) { return (w & 7) * G + (w >> 3); }

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
    int lo = 0, hi = s.B;  // the last b with cu[b] <= t
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

// value of one code
MOEB_DEV float kv_q4_value(uint32_t code, uint32_t sb) { return __fmaf_rn(bf16lo(sb), (float)code, bf16hi(sb)); }
MOEB_DEV float kv_fp4_value(uint32_t code) {
    const uint32_t m = code & 7u, e = m >> 1;
    const float v = 0.5f * (float)(e ? (2u + (m & 1u)) << (e - 1) : m);
    return (code & 8u) ? -v : v;
}
// 2^(byte - 127), NaN for 255
MOEB_DEV float kv_e8m0(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
// the 8 values of code word `word` (natural element order)
template <int FMT>
MOEB_DEV void kv_word_values(uint32_t word, uint32_t par, float (&o)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (FMT == FMT_Q4) o[i] = kv_q4_value((word >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u, par);
        else o[i] = kv_fp4_value((word >> (4 * i)) & 15u) * kv_e8m0(par);
    }
}
// parameters of word w of row `row` (int4: scale|bias; MXFP4: the E8M0 byte)
template <int FMT>
MOEB_DEV uint32_t kv_par(const void *ps, size_t row, int w, int D) {
    if (FMT == FMT_Q4) return static_cast<const uint32_t *>(ps)[row * (D / 64) + (w >> 3)];
    return static_cast<const uint8_t *>(ps)[row * (D / 32) + (w >> 2)];
}

struct KvWriteArgs {
    KvCache c;
    KvSeqs s;
    const uint16_t *k, *v;
    long k_row, k_head, v_row, v_head;  // strides in elements
};
struct KvReadArgs {
    KvCache c;
    KvSeqs s;          // s.lens = null: rows start at first[b] (null: 0)
    const int *first;
    uint16_t *k, *v;   // [T][Hkv][D]
};
struct KvAttnArgs {
    KvCache c;
    KvSeqs s;
    const uint16_t *q;
    long q_row, q_head;
    int H, Gq;         // query heads, query heads per KV head
    float scale;       // of the scores, times log2(e)
    int window, sinks;
    const float *sink_logits;  // [H] or null
    uint16_t *y;       // [T][H][D]
    float *lse;        // [T][H] or null
};
template <int FMT, int D>
__global__ void k_kv_write(KvWriteArgs a);
template <int FMT, int D>
__global__ void k_kv_read(KvReadArgs a);
template <int FMT, int D>
__global__ void k_kv_attn_rows(KvAttnArgs a);

}  // namespace moeb
