// Attention of many query rows per sequence over the 4-bit cache (prompts, and prompts' later pieces), on the
// 5th-generation tensor cores (layout of the cache: kv.cuh).
//
// A CTA takes 256 rows of one (sequence, KV head): the sequence's n tokens x Gq query heads in a row, as two tiles of 128
// (the tensor core's M), and walks the keys that any of them sees in tiles of 128, two halves of 64. Per half and row tile
//   S [128 x 64] = Q . K^T (operands in shared memory), P = 2^(S - m) as fp16 into the TMEM columns S leaves,
//   O [128 x D] += P . V (P from TMEM, V in shared memory, its D contiguous: the MN-major operand form).
// TMEM: O of both tiles (2 D columns), S / P of both tiles and halves (4 x 64). A row tile's products for one half run while
// its softmax is at the other half, and the two row tiles run side by side.
//   warps 0 - 15: softmax, two warpgroups per row tile: a thread has a row and 32 of a half's 64 keys, statistics in registers;
//     the two warps of 32 rows meet once per half, ask whether a row's maximum grew by more than 2^8 since it was last used
//     (P <= 2^14 in fp16 until then), and only then exchange the maxima and rescale O. (One thread per row leaves two such
//     warps per scheduler, too few to cover the waits between its steps: 4096-token prompt 200 us against 185. A thread with
//     all 64 keys of one half reads its scores twice and has to wait for the other half: 238 us.)
//   warps 16 - 19, 20 - 23: fetch the codes of K, of V (a tile ahead, in registers), dequantize them into fp16 tiles, 128-byte
//     swizzle
//   warps 24, 25: issue the products of row tile 0, 1 (26, 27 fill the warpgroup)
// Registers: 896 x 72 at launch; the softmax warpgroups go to 80, those of the products to 40 (64512 in all).
// Measured (int4 or MXFP4 within 2%; causal products counted once; calls in a row in a graph, call by call in brackets): 4096
// tokens of 32 heads on 4, D = 128: 183 (194) us, 750 TFLOP/s; 1000 rows of 64 heads on 32,001 keys of 8, D = 64: 955 (959) us,
// 540 TFLOP/s (its 2.0e9 exponentials need 433 us of their unit at 1965 MHz, 16 per SM and cycle; a quarter of them as
// polynomials on the FMA units gave nothing); 8191 tokens of 32 heads on 8 in a window of 2048 and 4 first tokens: 358 (366) us.
// Bound by the softmax warps: 65% to 67% of the issue slots are taken, 43% (D = 128) to 55% (D = 64) of the exponentials' unit, 39%
// to 27% of the tensor cores, and four such warps per scheduler do not cover all waits between a half's steps.
// fp16 and not bf16 operands: both formats' values, and P, would lose 2^-8 to bf16, as much as the result's own rounding;
// fp16 keeps 2^-11. Its range is kept by powers of two: one per query row, one per K tile (both go into the softmax's
// scale), and a running one for V (a change rescales O; it leaves room for 2^6 of growth, so that it hardly happens).
// A value that is NaN (a group that held one) must not reach rows that do not see its key, and 0 x NaN is NaN in a
// product: such a group enters as zeros, and the rows that see its key are marked and written as NaN. Likewise keys and
// queries, so that no score is NaN.
//
// Keys or values too far apart for the tile's power of two (KV_SPREAD) make the CTA's rows go through kv_exact as well, in fp32:
// the large ones may be later tokens', or have no weight, and would round the others away. Finding out costs 1% (4096 tokens 181
// -> 183 us); with values of ordinary models it does not happen (that prompt with such a token in every page: 41 ms).
//
// Every wait is bounded: after its limit the kernel records MOEB_DEVERR_TIMEOUT, its roles stop, TMEM is released.
#include "kv.cuh"

namespace moeb {

namespace {

constexpr int PR = 256;               // rows per CTA
constexpr int PT = 896;               // threads: seven warpgroups
constexpr float P_OFF = 6.f;          // P = 2^(score - m + 6)
constexpr float P_LAZY = 8.f;

template <int D>
struct Pr {
    static constexpr int C = D / 64;              // chunks of 64 values (128 bytes)
    static constexpr int NST = D == 128 ? 2 : 3;  // stages of K and of V
    static constexpr int TILE = C * 128 * 128;    // bytes of 128 rows
    static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + NST * TILE, BYTES = OFF_V + NST * TILE;
    static constexpr int SMEM = BYTES + 1024;
    static constexpr uint32_t S0 = 256;           // TMEM column of S
};

struct PrShared {
    uint64_t kfull[3], kempty[3], vfull[3], vempty[3], sfull[2][2], pfull[2][2], pv[2], ofull[2];  // [row tile][half]
    struct __align__(8) {
        float mul;             // 2^e of the K tile
        unsigned odd;          // byte per feeding warp: a key without a page or with a NaN among its own
    } k[4];                    // by key tile % 4
    unsigned hole[4][4], knan[4][4];  // those keys
    struct __align__(8) {
        float fix;             // what O is multiplied by before this V tile
        unsigned pz;           // byte per feeding warp: a NaN group among its rows
    } v[3];                    // by stage
    uint8_t pm[3][128];        // by stage and key: its NaN groups
    unsigned mx[2][2][4];      // exchange of the tiles' largest magnitudes: K or V, tile % 2, warp
    float qmul[PR];            // the rows' scale
    float rowx[2][PR];         // exchange between the two threads of a row
    float vun;                 // 2^e of O at the end
    uint32_t tmem;
    int b, tile, fail;
    int uneven;                // a group of K or V too far below the largest for fp16
};

MOEB_DEV float ex2p(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
MOEB_DEV float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
MOEB_DEV uint32_t h2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
MOEB_DEV uint32_t hmul2u(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
MOEB_DEV uint32_t hfma2u(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b), *reinterpret_cast<__half2 *>(&c));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// Waits for a phase, 2^22 tries at most. After that `fail` is set and every later wait returns soon: all roles go through their
// loops to the end (every address stays in bounds), so that none is left behind and TMEM is released. SLEEP: nanoseconds
// between the tries of a role that runs ahead of the others; its polling took a tenth of the issue slots.
template <int SLEEP = 0>
MOEB_DEV void pr_wait(uint32_t bar, unsigned parity, int *fail) {
    auto done = [&]() {
        unsigned ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok)
                     : "r"(bar), "r"(parity)
                     : "memory");
        return ok != 0;
    };
    if (done()) return;
#pragma unroll 1
    for (int n = 0; n < (SLEEP ? 1 << 14 : 1 << 12); ++n) {
#pragma unroll 1
        for (int i = 0; i < (SLEEP ? 256 : 1024); ++i) {
            if (done()) return;
            if (SLEEP) __nanosleep(SLEEP);
        }
        if (*reinterpret_cast<volatile int *>(fail)) return;
    }
    *reinterpret_cast<volatile int *>(fail) = 1;
}
template <int SLEEP = 0>
MOEB_DEV void pr_wait(uint64_t *bar, unsigned parity, int *fail) { pr_wait<SLEEP>(smem_u32(bar), parity, fail); }
// 128-byte swizzled operand descriptors: 8 rows of 128 bytes every 1024; LBO: bytes between 64-element chunks of an MN-major
// operand (K-major ones do not use it). The upper word is constant, the lower one is address / 16 and LBO / 16.
constexpr uint32_t DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
template <uint32_t LBO>
MOEB_DEV uint32_t desc_lo(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | (LBO >> 4) << 16; }
MOEB_DEV void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(DESC_HI)
        : "memory");
}
MOEB_DEV void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 db;\n mov.b64 db, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(DESC_HI)
        : "memory");
}
// one lane of a converged warp, the same one every time
MOEB_DEV bool elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
MOEB_DEV void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
MOEB_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
MOEB_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
MOEB_DEV void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
MOEB_DEV void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#define KV_R8(v, i) "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3]), "=f"(v[i + 4]), "=f"(v[i + 5]), "=f"(v[i + 6]), "=f"(v[i + 7])
// 32 columns of this warp's 32 lanes (issued only: wait_ld before use)
MOEB_DEV void ld32(uint32_t addr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : KV_R8(v, 0), KV_R8(v, 8), KV_R8(v, 16), KV_R8(v, 24)
        : "r"(addr));
}
#define KV_W8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
MOEB_DEV void ld16(uint32_t addr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : KV_R8(v, 0), KV_R8(v, 8)
        : "r"(addr));
}
MOEB_DEV void st16(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
                 KV_W8(v, 0), KV_W8(v, 8)
                 : "memory");
}

// The key tiles that rows at positions pmin .. pmax see: [0, ns) with the first tokens, then from lo / 128 on.
struct PrKeys {
    int lo, ns, nt;
};
MOEB_DEV PrKeys pr_keys(const KvAttnArgs &a, int pmin, int pmax) {
    PrKeys k;
    k.lo = a.window ? max(max(pmin, 0) - a.window + 1, 0) : 0;
    k.ns = min((min(a.sinks, k.lo) + 127) >> 7, k.lo >> 7);
    const int end = min(pmax + 1, a.s.P << a.c.pshift);  // of the keys: the last row's own, or the end of the page table
    k.nt = k.ns + max(((end + 127) >> 7) - (k.lo >> 7), 0);
    if (pmax < 0) k.ns = k.nt = 0;
    return k;
}
MOEB_DEV int pr_tok(const PrKeys &k, int i) { return (i < k.ns ? i : (k.lo >> 7) + i - k.ns) << 7; }

// a code word of 8 values to fp16, in the word's order; q4: s2 / b2 scale and bias, MXFP4: s2 / b2 the scales of the word's
// two half-words
template <int FMT>
MOEB_DEV uint4 pr_word(uint32_t w, uint32_t s2, uint32_t b2) {
    uint32_t o[4];
    if (FMT == FMT_Q4) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const uint32_t t = p & 2 ? w >> 8 : w;
            uint32_t v;
            if (p & 1) {  // 1024 + 16 q -> q
                asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(t), "r"(0x00F000F0u), "r"(0x64006400u));
                v = hfma2u(v, 0x2C002C00u, 0xD400D400u);  // 1 / 16, -64
            } else {      // 1024 + q -> q
                asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(t), "r"(0x000F000Fu), "r"(0x64006400u));
                const __half2 x = __hadd2(*reinterpret_cast<__half2 *>(&v), __float2half2_rn(-1024.f));
                v = *reinterpret_cast<const uint32_t *>(&x);
            }
            o[p] = hfma2u(v, s2, b2);
        }
    } else {
        asm("{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %4;\n cvt.rn.f16x2.e2m1x2 %0, b0;\n cvt.rn.f16x2.e2m1x2 %1, b1;\n"
            " cvt.rn.f16x2.e2m1x2 %2, b2;\n cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
            : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
            : "r"(w));
        o[0] = hmul2u(o[0], s2);
        o[1] = hmul2u(o[1], s2);
        o[2] = hmul2u(o[2], b2);
        o[3] = hmul2u(o[3], b2);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// the n lowest of 64 bits
MOEB_DEV unsigned long long pr_below(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

// bits 0, 4, 8 .. 28 as a byte
MOEB_DEV unsigned pr_byte(unsigned x) {
    x &= 0x11111111u;
    x = (x | x >> 3) & 0x03030303u;
    x = (x | x >> 6) & 0x000F000Fu;
    return (x | x >> 12) & 0xFFu;
}

// Largest magnitude (bits) that a row's parameters allow, NaN groups apart; nan: which groups are NaN; low: the smallest group's
// less KV_ZERO, groups below that wrapping to the top (they count as zeros).
template <int FMT, int NG>
MOEB_DEV uint32_t pr_top(const float (&s)[NG], const float (&b)[NG], unsigned &nan, uint32_t &low) {
    uint32_t top = 0;
    nan = 0;
    low = ~0u;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const float x = FMT == FMT_Q4 ? fmaxf(fabsf(b[g]), fabsf(fmaf(15.f, s[g], b[g]))) : 6.f * s[g];
        const uint32_t u = __float_as_uint(x);
        if (u < 0x7f800000u && s[g] == s[g]) {
            top = max(top, u);
            low = min(low, u - KV_ZERO);
        } else {
            nan |= 1u << g;
        }
    }
    return top;
}

// One warpgroup's work on K or V: every key tile's codes to fp16 in its stage. Warp w has keys 32 i + 8 w + r, r = lane / 4, in
// four passes i, a lane a quarter of each row; lane (r, c) is the owner of key 32 c + 8 w + r: it looks up the page, reads the
// parameters and prepares them for all, the passes take them by shuffles. Codes are on their way a tile ahead, parameters and
// page ids two. One body for K and V: five kinds of warps share the instruction cache.
template <int FMT, int D>
MOEB_DEV void pr_feed(const KvAttnArgs &a, PrShared &sh, unsigned char *sm, const PrKeys &keys, int b, int h, int k0, int nk, int pmax,
                      int w, int lane, bool V) {
    using L = Pr<D>;
    constexpr int NST = L::NST, W4 = D / 32, NG = FMT == FMT_Q4 ? D / 64 : D / 32, NP = FMT == FMT_Q4 ? NG : 1;
    constexpr int PB = FMT == FMT_Q4 ? 4 * NG : NG;  // parameter bytes per row
    const int r = lane >> 2, c = lane & 3, mine = 32 * c + 8 * w + r;
    const unsigned char *codes = reinterpret_cast<const unsigned char *>(V ? a.c.vq : a.c.kq) + ((size_t)h << a.c.pshift) * (D / 2) + c * (D / 8);
    const unsigned char *pars = static_cast<const unsigned char *>(V ? a.c.vs : a.c.ks) + ((size_t)h << a.c.pshift) * PB;
    const size_t per_page = (size_t)a.c.Hkv << a.c.pshift;  // rows
    const int *table = a.s.table + (size_t)b * a.s.trow;
    const int pmask = (1 << a.c.pshift) - 1;
    uint64_t *full = V ? sh.vfull : sh.kfull, *empty = V ? sh.vempty : sh.kempty;
    unsigned char *dst0 = sm + (V ? L::OFF_V : L::OFF_K) + (8 * w + r) * 128;
    uint32_t code[4][W4], par[NP];
    // page id of this lane's key of tile k: -1 where no row sees the key, -2 where it has no page
    auto page = [&](int k) {
        const int j = pr_tok(keys, k0 + k) + mine;
        if (k >= nk || j > pmax || (j < keys.lo && j >= a.sinks)) return -1;
        const int pi = j >> a.c.pshift, id = pi < a.s.P ? table[pi] : -1;
        return id < 0 || id >= a.c.pages ? -2 : id;
    };
    auto fetch_par = [&](int k, int id) {
#pragma unroll
        for (int x = 0; x < NP; ++x) par[x] = 0u;
        if (id < 0) return;
        const unsigned char *p = pars + (id * per_page + (size_t)((pr_tok(keys, k0 + k) + mine) & pmask)) * PB;
        if (PB == 8) {
            const uint2 x = *reinterpret_cast<const uint2 *>(p);
            par[0] = x.x;
            par[NP - 1] = x.y;
        } else if (PB == 4) {
            par[0] = *reinterpret_cast<const uint32_t *>(p);
        } else {
            par[0] = *reinterpret_cast<const uint16_t *>(p);
        }
    };
    auto fetch_codes = [&](int k, int id) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pid = __shfl_sync(0xffffffffu, id, (lane & 28) | i);
#pragma unroll
            for (int x = 0; x < W4; ++x) code[i][x] = 0u;
            if (pid >= 0) {
                const unsigned char *p = codes + (pid * per_page + (size_t)((pr_tok(keys, k0 + k) + 32 * i + 8 * w + r) & pmask)) * (D / 2);
                if (D == 128) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(p);
                    code[i][0] = x.x; code[i][1] = x.y; code[i][W4 - 2] = x.z; code[i][W4 - 1] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2 *>(p);
                    code[i][0] = x.x; code[i][1] = x.y;
                }
            }
        }
    };
    int id = page(0), id1 = page(1);
    fetch_par(0, id);
    fetch_codes(0, id);
    uint32_t vlim = 0;  // V: bits of the largest value that the running power of two takes; that power, its inverse
    float vmul = 1.f, vun = 1.f;
    int st = 0;
    unsigned ph = 1;
#pragma unroll 1
    for (int j = 0; j < nk; ++j) {
        // ---- this lane's key: the largest magnitude its parameters allow, its NaN groups
        float s[NG], bb[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            s[g] = FMT == FMT_Q4 ? bf16lo(par[FMT == FMT_Q4 ? g : 0]) : kv_e8m0((par[0] >> (8 * g)) & 255u);
            bb[g] = FMT == FMT_Q4 ? bf16hi(par[FMT == FMT_Q4 ? g : 0]) : 0.f;
        }
        unsigned nan;
        uint32_t low, top = pr_top<FMT, NG>(s, bb, nan, low);
        if (id < 0) top = 0, low = ~0u;  // zeros (MXFP4: codes of zero)
        const unsigned hole = __ballot_sync(0xffffffffu, id == -2);
        id = id1;
        fetch_par(j + 1, id);  // of the next tile; what this one needs is in s and bb
        id1 = page(j + 2);
        top = __reduce_max_sync(0xffffffffu, top);
        unsigned *mx = sh.mx[V][j & 1];
        if (lane == 0) mx[w] = top;
        asm volatile("bar.sync %0, 128;" ::"r"(V ? 2 : 1) : "memory");
        top = max(max(mx[0], mx[1]), max(mx[2], mx[3]));
        if (j >= NST) pr_wait<100>(empty + st, ph, &sh.fail);
        {
            // ---- the tile's power of two
            float mul, fix = 1.f;
            if (!V || top > vlim) {
                const uint32_t e = min(max(top >> 23, 9u), 248u);
                const float nm = __uint_as_float((262u - e) << 23), nu = __uint_as_float((e - 8u) << 23);
                fix = nm * vun;
                vmul = nm;
                vun = nu;
                vlim = (e + 6u) << 23;
            }
            mul = vmul;
            if (low < (uint32_t)max((int)vlim - ((KV_SPREAD + 6) << 23) - (int)KV_ZERO, 0)) sh.uneven = 1;
            uint32_t s2[NG], b2[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if ((nan >> g) & 1u) s[g] = bb[g] = 0.f;  // the rows that see the key are marked instead
                s2[g] = h2(s[g] * mul, s[g] * mul);
                b2[g] = h2(bb[g] * mul, bb[g] * mul);
            }
            unsigned char *dst = dst0 + st * L::TILE;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t ps[NG], pb[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    ps[g] = __shfl_sync(0xffffffffu, s2[g], (lane & 28) | i);
                    pb[g] = FMT == FMT_Q4 ? __shfl_sync(0xffffffffu, b2[g], (lane & 28) | i) : 0u;
                }
#pragma unroll
                for (int x = 0; x < W4; ++x) {
                    const int u = c * W4 + x;
                    const uint4 v = FMT == FMT_Q4 ? pr_word<FMT>(code[i][x], ps[x % NG], pb[x % NG])
                                                  : pr_word<FMT>(code[i][x], ps[(2 * x) % NG], ps[(2 * x + 1) % NG]);
                    *reinterpret_cast<uint4 *>(dst + (u >> 3) * 16384 + i * 4096 + (((u & 7) ^ r) << 4)) = v;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            // ---- what the softmax has to know of the tile
            if (V) {
                const bool any = __any_sync(0xffffffffu, nan != 0);
                if (any) sh.pm[st][mine] = (uint8_t)nan;
                if (lane == 0) {
                    reinterpret_cast<uint8_t *>(&sh.v[st].pz)[w] = any;
                    if (w == 0) {
                        sh.v[st].fix = fix;
                        sh.vun = vun;
                    }
                }
            } else {
                const unsigned bad = __ballot_sync(0xffffffffu, nan != 0);
                if (lane < 4) {  // byte w of word `lane`: keys 32 lane + 8 w .., their bits are 4 r + lane
                    const unsigned x = pr_byte(hole >> lane);
                    reinterpret_cast<uint8_t *>(sh.hole[j & 3])[4 * lane + w] = (uint8_t)x;
                    reinterpret_cast<uint8_t *>(sh.knan[j & 3])[4 * lane + w] = (uint8_t)pr_byte(bad >> lane);
                    if (x) atomicOr(a.c.err, ERR_PAGE);
                }
                if (lane == 0) {
                    reinterpret_cast<uint8_t *>(&sh.k[j & 3].odd)[w] = (hole | bad) != 0;
                    if (w == 0) sh.k[j & 3].mul = vun;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(full + st);
        }
        fetch_codes(j + 1, id);
        if (++st == NST) {
            st = 0;
            ph ^= 1;
        }
    }
}

// The products of row tile T. The whole warp goes along and one lane issues: what the instructions take (addresses, counts)
// is the warp's own, so that it sits in uniform registers; a lane on its own needs 150 cycles to issue a product.
template <int D, int T>
MOEB_DEV void pr_products(const KvAttnArgs &a, PrShared &sh, unsigned char *sm, int nk_, uint32_t tmem_) {
    using L = Pr<D>;
    constexpr int NST = L::NST;
    constexpr uint32_t id_s = (1u << 4) | (8u << 17) | (8u << 24);
    constexpr uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
    const int nk = __shfl_sync(0xffffffffu, nk_, 0);
    if (nk == 0) return;
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_, 0), base = __shfl_sync(0xffffffffu, smem_u32(sm), 0);
    const uint32_t ds = tmem + L::S0 + 128 * T, dout = tmem + D * T;
    const uint32_t qa = desc_lo<16>(base + T * L::TILE), ka0 = desc_lo<16>(base + L::OFF_K), va0 = desc_lo<16384>(base + L::OFF_V);
    // S of half i of key tile j (stage st, phase ph); the last product of K's stage frees it
    auto scores = [&](int st, unsigned ph, int i) {
        if (i == 0) pr_wait(sh.kfull + st, ph, &sh.fail);
        fence_after();
        const uint32_t ka = ka0 + (st * L::TILE + i * 8192) / 16;
        if (elect()) {
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
                const uint32_t off = ((s >> 2) * 16384 + (s & 3) * 32) / 16;
                mma_ss(ds + 64 * i, qa + off, ka + off, id_s, s > 0);
            }
            commit(&sh.sfull[T][i]);
            if (i) commit(sh.kempty + st);
        }
        __syncwarp();
    };
    scores(0, 0, 0);
    scores(0, 0, 1);
    int st = 0, sn = NST > 1 ? 1 : 0;  // stage of this tile and of the next, with their phases
    unsigned ph = 0, pn = 0;
#pragma unroll 1
    for (int j = 0; j < nk; ++j) {
        const uint32_t va = va0 + st * (L::TILE / 16);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i == 0) pr_wait(sh.vfull + st, ph, &sh.fail);
            pr_wait<40>(&sh.pfull[T][i], j & 1, &sh.fail);
            fence_after();
            if (elect()) {
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    mma_ts(dout, ds + 64 * i + 8 * s, va + (i * 8192 + s * 2048) / 16, id_o, i > 0 || s > 0 ? 1u : (j > 0));
                commit(sh.pv + T);
                if (i) commit(sh.vempty + st);
            }
            __syncwarp();
            if (j + 1 < nk) scores(sn, pn, i);
        }
        st = sn;
        ph = pn;
        if (++sn == NST) {
            sn = 0;
            pn ^= 1;
        }
    }
    if (elect()) commit(sh.ofull + T);
    __syncwarp();
    int own = 0;
    pr_wait(sh.ofull + T, 0, &own);  // nothing is in flight when TMEM is released, after a failure either
}

}  // namespace

// part: null, or the workspace of split calls: [splits][T][H][D] sums, then [splits][T][H] (max, sum)
template <int FMT, int D>
__global__ void __launch_bounds__(PT, 1) k_kv_attn_prompt(const KvAttnArgs a, int tiles, float *part) {
    using L = Pr<D>;
    constexpr int NST = L::NST, NG = FMT == FMT_Q4 ? D / 64 : D / 32;
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    __shared__ PrShared sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int h = blockIdx.x % a.c.Hkv;
    pdl_wait();
    // ---- the sequence of this row tile; the last tiles of a sequence see the most keys and come first
    if (warp == 0) {
        const int gt = tiles - 1 - (int)(blockIdx.x / a.c.Hkv);
        int b = -1, at = 0;
        if (!a.s.cu) {
            const int per = (int)(((long)a.s.each * a.Gq + PR - 1) / PR);
            b = gt / per;
            at = gt - b * per;
        } else {
            int base = 0;
            for (int i = 0; i < a.s.B && b < 0; i += 32) {
                int n = 0;
                if (i + lane < a.s.B) {
                    int r0, r1;
                    kv_rows(a.s, i + lane, r0, r1);
                    const long c = (long)(r1 - r0) * a.Gq;
                    n = c <= a.few ? 0 : (int)((c + PR - 1) / PR);
                }
                int inc = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += v;
                }
                const unsigned m = __ballot_sync(0xffffffffu, base + inc > gt);
                if (m) {
                    const int l = __ffs(m) - 1;
                    b = i + l;
                    at = gt - base - (__shfl_sync(0xffffffffu, inc, l) - __shfl_sync(0xffffffffu, n, l));
                }
                base += __shfl_sync(0xffffffffu, inc, 31);
            }
        }
        if (lane == 0) {
            sh.b = b;
            sh.tile = at;
            sh.fail = sh.uneven = 0;
        }
    }
    __syncthreads();
    const int b = sh.b;
    if (b < 0) return;
    int r0, r1;
    kv_rows(a.s, b, r0, r1);
    const int n = r1 - r0, Lk = max(a.s.lens[b], 0), R0 = sh.tile * PR, NR = n * a.Gq;
    const int p0 = Lk - n;  // position of row 0
    const int pmin = p0 + R0 / a.Gq, pmax = p0 + (min(R0 + PR, NR) - 1) / a.Gq;
    const PrKeys keys = pr_keys(a, pmin, pmax);
    if (threadIdx.x == 0 && pmax >= a.s.P << a.c.pshift) atomicOr(a.c.err, ERR_PAGE);  // tokens that the table has no place for
    const int ns = gridDim.y, sp = blockIdx.y;
    const int k0 = (int)((long)keys.nt * sp / ns), k1 = (int)((long)keys.nt * (sp + 1) / ns), nk = k1 - k0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NST; ++i) {
            mbar_init(sh.kfull + i, 4);
            mbar_init(sh.kempty + i, 2);
            mbar_init(sh.vfull + i, 4);
            mbar_init(sh.vempty + i, 2);
        }
        for (int i = 0; i < 2; ++i) {
            for (int x = 0; x < 2; ++x) {
                mbar_init(&sh.sfull[i][x], 1);
                mbar_init(&sh.pfull[i][x], 8);
            }
            mbar_init(sh.pv + i, 1);
            mbar_init(sh.ofull + i, 1);
        }
        mbar_fence_init();
        sh.vun = 1.f;
    }
    if (warp == 24) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // ---- queries: fp16 after a power of two per row (the largest value near 2^8), K's order of values (kv_dim; V's columns of O
    // keep it too), swizzled. D / 8
    // lanes have a row (one word of 8 values each), so that the loads are whole lines.
    if (warp < 16) {
        constexpr int LR = D / 8, RW = 32 / LR;  // lanes per row, rows per load
        const int x = lane % LR;
        uint4 w[16 / RW];
#pragma unroll
        for (int i = 0; i < 16 / RW; ++i) {
            const int R = R0 + warp * 16 + i * RW + lane / LR;
            w[i] = make_uint4(0, 0, 0, 0);
            if (R < NR) {
                const int ri = R / a.Gq;
                const uint16_t *src = a.q + (r0 + ri) * a.q_row + (h * a.Gq + R - ri * a.Gq) * a.q_head;
                const uint2 lo = *reinterpret_cast<const uint2 *>(src + kv_dim<FMT, D>(2 * x));
                const uint2 hi = *reinterpret_cast<const uint2 *>(src + kv_dim<FMT, D>(2 * x + 1));
                w[i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
            }
        }
#pragma unroll
        for (int i = 0; i < 16 / RW; ++i) {
            const int row = warp * 16 + i * RW + lane / LR;
            const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(u[e] & 0x7fffu, (u[e] >> 16) & 0x7fffu));
#pragma unroll
            for (int e = 1; e < LR; e <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, e));
            const int e = min(max((int)(top >> 7), 9), 254);
            float down = __uint_as_float((uint32_t)(262 - e) << 23);
            float qmul = fabsf(a.scale) * __uint_as_float((uint32_t)(e - 8) << 23);
            if (a.scale < 0.f) down = -down;  // the softmax's scale stays positive: it takes the maximum before scaling
            if (a.scale == 0.f) down = 0.f, qmul = 1.f;
            const bool fine = top < 0x7f80u;
            uint32_t o[4];
#pragma unroll
            for (int e2 = 0; e2 < 4; ++e2) o[e2] = fine ? h2(bf16lo(u[e2]) * down, bf16hi(u[e2]) * down) : 0u;
            if (!fine) qmul = -1.f;  // an infinity or a NaN in the row: its result is NaN
            *reinterpret_cast<uint4 *>(sm + (row >> 7) * L::TILE + (x >> 3) * 16384 + (row & 127) * 128 + (((x & 7) ^ (row & 7)) << 4)) =
                make_uint4(o[0], o[1], o[2], o[3]);
            if (x == 0) sh.qmul[row] = qmul;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp >= 24) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        // ------------------------------------------------------------ products, a warp per row tile
        if (warp == 24) pr_products<D, 0>(a, sh, sm, nk, tmem);
        if (warp == 25) pr_products<D, 1>(a, sh, sm, nk, tmem);
    } else if (warp >= 16) {
        // ------------------------------------------------------------ codes -> fp16 tiles, K or V
        pr_feed<FMT, D>(a, sh, sm, keys, b, h, k0, nk, pmax, warp & 3, lane, warp >= 20);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 80;");
        // ------------------------------------------------------------ softmax of row tile t: two threads per row (sub)
        const int t = warp >> 3, sub = (warp >> 2) & 1, row = (warp & 3) * 32 + lane, R = R0 + t * 128 + row;
        const bool have = R < NR;
        const int ri = R / a.Gq, pos = have ? p0 + ri : -1, row_t = have ? r0 + ri : 0, row_h = h * a.Gq + R - ri * a.Gq;
        const float qmul = sh.qmul[t * 128 + row];
        unsigned poison = qmul < 0.f ? 1u << 31 : 0u;  // bit g: group g of the row is NaN; bit 31: all of it
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + L::S0 + 128 * t, to = tmem + lanes + D * t + sub * (D / 2);
        const int meet = 3 + 4 * t + (warp & 3);  // barrier of the two warps that have the same rows
        auto meet_any = [&](bool mine) {  // true for one of the two warps' threads
            unsigned r;
            asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, 64, p;\n selp.u32 %0, 1, 0, q;\n}"
                         : "=r"(r) : "r"((unsigned)mine), "r"(meet) : "memory");
            return r != 0;
        };
        auto other = [&](float mine) {  // the row's other thread's value; the threads meet again before the next exchange
            sh.rowx[sub][t * 128 + row] = mine;
            asm volatile("bar.sync %0, 64;" ::"r"(meet) : "memory");
            return sh.rowx[sub ^ 1][t * 128 + row];
        };
        const int q0 = R0 + t * 128;
        const int tmin = p0 + q0 / a.Gq, tmax = p0 + (min(q0 + 128, NR) - 1) / a.Gq;  // positions of the tile's rows
        // m: what the weights are relative to; a row that has seen no key yet has the lowest number and no weight
        constexpr float LOW = -3e38f;
        float m = LOW, sc = 0.f;
        uint64_t l2 = 0;  // two partial sums of the weights
        int st = 0, j0 = pr_tok(keys, k0);
        unsigned vph = 0, par = 0;
        // every row sees all of a half from j0 on: j0 <= jf, and j0 > jw or j0 <= js
        const int jf = tmin - 63, jw = a.window ? tmax - a.window : -1, js = a.window ? a.sinks - 64 : -1;
        const uint32_t sf = smem_u32(&sh.sfull[t][0]), pf = smem_u32(&sh.pfull[t][0]), vf = smem_u32(sh.vfull);
#pragma unroll 1
        for (int j = 0; j < nk; ++j) {
            unsigned odd = 0;
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
                pr_wait(sf + 8 * i2, par, &sh.fail);
                fence_after();
                float v[32];
                ld32(ts + 64 * i2 + 32 * sub, v);
                float vfix = 1.f;
                if (i2 == 0) {
                    sc = fmaxf(fabsf(qmul) * sh.k[j & 3].mul, 1.2e-38f);  // above zero: a hidden score of -inf stays -inf
                    odd = sh.k[j & 3].odd;
                    // V's stage: its power of two, its NaN groups
                    pr_wait(vf + 8 * st, vph, &sh.fail);
                    vfix = sh.v[st].fix;
                    if (const unsigned pz = sh.v[st].pz) {
#pragma unroll 1
                        for (int e = 0; e < 128; ++e) {
                            if (!((pz >> (8 * ((e >> 3) & 3))) & 1u)) continue;
                            const unsigned g = sh.pm[st][e];
                            if (g && e <= pos - j0 && (!a.window || e > pos - a.window - j0 || e < a.sinks - j0)) poison |= g;
                        }
                        __syncwarp();
                    }
                }
                wait_ld();
                if (!(j0 <= jf && (j0 > jw || j0 <= js)) || odd) {
                    // bit i: this row sees key i of the half
                    const unsigned long long hole = (unsigned long long)sh.hole[j & 3][2 * i2 + 1] << 32 | sh.hole[j & 3][2 * i2];
                    const unsigned long long old = a.window ? pr_below(pos - a.window + 1 - j0) & ~pr_below(a.sinks - j0) : 0ull;
                    const unsigned long long see = pr_below(pos - j0 + 1) & ~old & ~hole;
                    const unsigned s0 = (unsigned)see, s1 = (unsigned)(see >> 32), mine = sub ? s1 : s0;
                    if (odd && ((s0 & sh.knan[j & 3][2 * i2]) | (s1 & sh.knan[j & 3][2 * i2 + 1]))) poison |= 1u << 31;
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = (mine >> i) & 1u ? v[i] : -INFINITY;
                }
                j0 += 64;
                float x0 = max3(v[0], v[1], v[2]), x1 = max3(v[3], v[4], v[5]), x2 = max3(v[6], v[7], v[8]), x3 = max3(v[9], v[10], v[11]);
#pragma unroll
                for (int i = 12; i < 28; i += 8) {
                    x0 = max3(x0, v[i], v[i + 1]);
                    x1 = max3(x1, v[i + 2], v[i + 3]);
                    x2 = max3(x2, v[i + 4], v[i + 5]);
                    x3 = max3(x3, v[i + 6], v[i + 7]);
                }
                const float top = max3(max3(x0, v[28], v[29]), max3(x1, v[30], v[31]), fmaxf(x2, x3));
                // rescale O when a maximum of the two warps' rows grew far, or V's power of two changed. Both have read their
                // scores when they meet: P may take their columns
                if (meet_any(top * sc > m + P_LAZY || (i2 == 0 && vfix != 1.f))) {
                    const float mt = fmaxf(top, other(top)) * sc;
                    float ff = vfix;
                    if (mt > m + P_LAZY) {
                        if (mt == INFINITY) poison |= 1u << 31;  // a score past fp32: inf - inf
                        const float f = ex2p(m - mt);
                        m = mt;
                        l2 = mul2(l2, pair(f, f));
                        ff *= f;
                    }
                    if (j > 0 || i2 > 0) {
                        pr_wait(sh.pv + t, i2 ^ 1, &sh.fail);  // the half before: phase 2 j + i2 - 1
                        fence_after();
#pragma unroll 1
                        for (int x = 0; x < D / 2; x += 16) {
                            float o[16];
                            __syncwarp();
                            ld16(to + x, o);
                            wait_ld();
                            uint32_t u[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(o[i] * ff);
                            st16(to + x, u);
                        }
                    }
                }
                const float off = P_OFF - m;
                const uint64_t sc2 = pair(sc, sc), off2 = pair(off, off);
                uint32_t u[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x, y;
                    unpair(fma2(pair(v[2 * i], v[2 * i + 1]), sc2, off2), x, y);
                    x = ex2p(x);
                    y = ex2p(y);
                    l2 = add2(l2, pair(x, y));
                    u[i] = h2(x, y);
                }
                st16(ts + 64 * i2 + 16 * sub, u);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pf + 8 * i2) : "memory");
            }
            par ^= 1;
            if (++st == NST) {
                st = 0;
                vph ^= 1;
            }
            if (k0 + j + 1 == keys.ns) j0 = pr_tok(keys, keys.ns);
        }
        if (nk > 0) pr_wait(sh.ofull + t, 0, &sh.fail);
        fence_after();
        __syncwarp();
        float l;
        {  // the row's sum: both threads add in the same order
            float la, lb;
            unpair(l2, la, lb);
            const float mine = la + lb, o = other(mine);
            l = sub ? o + mine : mine + o;
        }
        if (poison >> 31 && (qmul >= 0.f || l != 0.f)) l = __uint_as_float(0x7fffffffu);  // a query that sees nothing is not looked at
        // ---- the rows' results (m is off by P_OFF against the weights' sum: undone here)
        const float M = l == 0.f ? -INFINITY : m - P_OFF;
        // a tile with groups too far apart for fp16 (the feeders set the mark before their tiles were full), or scores that are too
        // large, the same for both warps of the rows: these go through kv_exact below
        const bool again = *reinterpret_cast<volatile int *>(&sh.uneven) || __any_sync(0xffffffffu, fabsf(m) > KV_FAR && m != LOW);
        float mul = nk > 0 ? sh.vun : 0.f, Ls = l, sum_m = M;
        if (!part) {
            if (a.sink_logits && have) {
                const float s = a.sink_logits[row_h] * 1.4426950408889634f, N = fmaxf(M, s), use = N == -INFINITY ? 0.f : N;
                const float f = exp2f(M - use);
                mul *= f;
                Ls = Ls * f + exp2f(s - use);
                sum_m = N;
            }
            mul = Ls == 0.f ? 0.f : mul / Ls;
        }
        const size_t orow = (size_t)row_t * a.H + row_h;
        // bf16 rows go through the tile's place of Q (its products are over), so that the stores are whole lines.
        unsigned char *stage = sm + t * L::TILE + (warp & 3) * (32 * D * 2);
        float *pd = part ? part + ((size_t)sp * a.s.T * a.H + orow) * D : nullptr;
#pragma unroll
        for (int x = 0; x < D / 2; x += 32) {
            float o[32];
            if (nk > 0) {
                ld32(to + x, o);
                wait_ld();
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const int d = sub ? kv_dim<FMT, D>((D / 2 + x + i) / 4) : kv_dim<FMT, D>((x + i) / 4), g = d / (FMT == FMT_Q4 ? 64 : 32);
                float y[4];
                const bool nanv = (poison >> g) & 1u;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = nanv ? __uint_as_float(0x7fffffffu) : mul == 0.f && l == 0.f ? 0.f : o[i + e] * mul;
                if (!part) {
                    *reinterpret_cast<uint2 *>(stage + lane * (D * 2) + (((d >> 3) ^ (lane & 7)) << 4) + (d & 4) * 2) =
                        make_uint2(pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]));
                } else if (have) {
                    *reinterpret_cast<float4 *>(pd + d) = make_float4(y[0], y[1], y[2], y[3]);
                }
            }
            __syncwarp();
        }
        if (!part) {
            constexpr int LR = D / 8, RW = 32 / LR;
            asm volatile("bar.sync %0, 64;" ::"r"(meet) : "memory");
#pragma unroll 4
            for (int i = 16 * sub; i < 16 * sub + 16; i += RW) {
                const int rr = i + lane / LR, x = lane % LR, Rr = R0 + t * 128 + (warp & 3) * 32 + rr;
                if (Rr < NR && !again) {  // y may lie where q does, which kv_exact reads
                    const int ri2 = Rr / a.Gq;
                    const uint4 v = *reinterpret_cast<const uint4 *>(stage + rr * (D * 2) + ((x ^ (rr & 7)) << 4));
                    *reinterpret_cast<uint4 *>(a.y + ((size_t)(r0 + ri2) * a.H + h * a.Gq + Rr - ri2 * a.Gq) * D + 8 * x) = v;
                }
            }
        }
        if (have && sub == 0) {
            if (part) reinterpret_cast<float2 *>(part + (size_t)ns * a.s.T * a.H * D)[(size_t)sp * a.s.T * a.H + orow] = make_float2(M, l);
            else if (a.lse) a.lse[orow] = Ls == 0.f ? -INFINITY : (sum_m + log2f(Ls)) * 0.6931471805599453f;
        }
        fence_before();
        // ---- the rows that are this warp's to store once more, in fp32. No barrier below: after a timeout one warp of the rows may
        // have found the mark and the other not
        asm volatile("bar.sync %0, 64;" ::"r"(meet) : "memory");
        if (again) {
            const int Ru = R0 + t * 128 + (warp & 3) * 32 + 16 * sub;
#pragma unroll 1
            for (int i = 0; i < 16 && Ru + i < NR; ++i) {
                const int xi = (Ru + i) / a.Gq, xh = h * a.Gq + Ru + i - xi * a.Gq;
                const KvSum x = kv_exact<FMT, D>(a, b, h, a.q + (r0 + xi) * a.q_row + xh * a.q_head, p0 + xi, k0, k1, keys.ns, (keys.lo >> 7) - keys.ns);
                if (lane >= D / 4) continue;
                const size_t xrow = (size_t)(r0 + xi) * a.H + xh;
                if (!part) {
                    kv_finish<D>(a, r0 + xi, xh, kv_dim<FMT, D>(lane) / 4, x.v, x.M, x.L);
                    continue;
                }
                *reinterpret_cast<float4 *>(part + ((size_t)sp * a.s.T * a.H + xrow) * D + kv_dim<FMT, D>(lane)) = x.v;
                if (lane == 0)
                    reinterpret_cast<float2 *>(part + (size_t)ns * a.s.T * a.H * D)[(size_t)sp * a.s.T * a.H + xrow] = make_float2(x.M, x.L);
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && sh.fail) atomicOr(a.c.err, ERR_TIMEOUT);
    if (warp == 24) {
        __syncwarp();
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Joins the partial sums of a call whose keys were split: a warp per (row, head).
template <int D>
__global__ void __launch_bounds__(128) k_kv_attn_join_splits(const KvAttnArgs a, const float *part, int ns) {
    pdl_wait();
    const size_t rows = (size_t)a.s.T * a.H, row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int t = (int)(row / a.H), lane = threadIdx.x & 31;
    int r0, r1;
    const int b = kv_seq_of(a.s, t, r0, r1);
    if (b < 0 || (long)(r1 - r0) * a.Gq <= a.few || lane >= D / 4) return;
    const float2 *ml = reinterpret_cast<const float2 *>(part + (size_t)ns * rows * D);
    float M = -INFINITY, S = 0.f;
    for (int i = 0; i < ns; ++i) M = fmaxf(M, ml[i * rows + row].x);
    const float use = M == -INFINITY ? 0.f : M;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < ns; ++i) {
        const float2 x = ml[i * rows + row];
        const float f = ex2p(x.x - use);
        const float4 w = *reinterpret_cast<const float4 *>(part + (i * rows + row) * D + 4 * lane);
        S += x.y * f;
        v.x += w.x * f;
        v.y += w.y * f;
        v.z += w.z * f;
        v.w += w.w * f;
    }
    kv_finish<D>(a, t, (int)(row - (size_t)t * a.H), lane, v, M, S);
}

size_t kv_prompt_smem(int D) { return D == 128 ? Pr<128>::SMEM : Pr<64>::SMEM; }

template __global__ void k_kv_attn_prompt<FMT_Q4, 64>(const KvAttnArgs, int, float *);
template __global__ void k_kv_attn_prompt<FMT_Q4, 128>(const KvAttnArgs, int, float *);
template __global__ void k_kv_attn_prompt<FMT_FP4, 64>(const KvAttnArgs, int, float *);
template __global__ void k_kv_attn_prompt<FMT_FP4, 128>(const KvAttnArgs, int, float *);
template __global__ void k_kv_attn_join_splits<64>(const KvAttnArgs, const float *, int);
template __global__ void k_kv_attn_join_splits<128>(const KvAttnArgs, const float *, int);

}  // namespace moeb
