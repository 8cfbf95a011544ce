// Attention of many query rows per sequence over the 4-bit cache (prompts, and prompts' later pieces), on the
// 5th-generation tensor cores (layout of the cache: kv.cuh).
//
// A CTA takes 256 rows of one (sequence, KV head): the sequence's n tokens x Gq query heads in a row, as two tiles of 128
// (the tensor core's M), and walks the keys that any of them sees in tiles of 128. Per key tile and row tile
//   S [128 x 128] = Q . K^T (operands in shared memory), P = 2^(S - m) as fp16 into the TMEM columns S leaves,
//   O [128 x D] += P . V (P from TMEM, V in shared memory, its D contiguous: the MN-major operand form).
// TMEM: O of both tiles (2 D columns), S / P of both tiles (2 x 128). While one row tile is in its softmax the other one's
// products run, so the tensor core and the exponentials work side by side.
//   warps 0 - 3, 4 - 7: softmax of row tile 0, 1: a thread per row, statistics in registers; they also rescale O, only when
//     a row's maximum grew by more than 2^8 since it was last used (P <= 2^14 in fp16 until then)
//   warps 8 - 11: fetch codes (a tile ahead, in registers), dequantize K and V into fp16 tiles, 128-byte swizzle
//   warps 12, 13: one lane each issues the products of row tile 0, 1 (14, 15 fill the warpgroup)
// Registers: 512 x 128 at launch; the softmax warpgroups go to 160, the others to 120 and 56 (63488 of 65536 in all).
// fp16 and not bf16 operands: both formats' values, and P, would lose 2^-9 to bf16, as much as the result's own rounding;
// fp16 keeps 2^-12. Its range is kept by powers of two: one per query row, one per K tile (both go into the softmax's
// scale), and a running one for V (a change rescales O; it leaves room for 2^6 of growth, so that it hardly happens).
// A value that is NaN (a group that held one) must not reach rows that do not see its key, and 0 x NaN is NaN in a
// product: such a group enters as zeros, and the rows that see its key are marked and written as NaN.
//
// Every wait is bounded: after its limit the kernel records MOEB_DEVERR_TIMEOUT, its roles stop, TMEM is released.
#include <cuda_fp16.h>

#include "kv.cuh"

namespace moeb {

namespace {

constexpr int PR = 256;               // rows per CTA
constexpr int PT = 512;               // threads: four warpgroups
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
    uint64_t kfull[3], kempty[3], vfull[3], vempty[3], sfull[2], pfull[2], ofull[2];
    float kmul[4];             // by key tile % 4: 2^e of the K tile
    unsigned hole[4][4];       // by key tile % 4: keys without a page
    float vfix[3];             // by stage: what O is multiplied by before this V tile
    unsigned pz[3];            // by stage: byte per dequantizing warp, a NaN group among its rows
    uint8_t pm[3][128];        // by stage and key: its NaN groups
    unsigned mx[2][4][2];      // exchange of the tile's largest magnitudes
    float vun;                 // 2^e of O at the end
    uint32_t tmem;
    int b, tile, fail;
};

MOEB_DEV float ex2p(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
// Waits for a phase, at most 2 s of wall time or until another role has given up.
MOEB_DEV bool pr_wait(uint64_t *bar, unsigned parity, const int *fail) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (unsigned i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 31u) == 0 && (*reinterpret_cast<const volatile int *>(fail) || globaltimer_ns() - t0 > 2000000000ull)) return false;
    }
}
// 128-byte swizzled operand descriptor: 8 rows of 128 bytes every 1024; lbo: bytes between 64-element chunks of an MN-major
// operand (K-major ones do not use it)
MOEB_DEV uint64_t sdesc(uint32_t saddr, uint32_t lbo) {
    uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(lbo >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
MOEB_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a),
        "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
MOEB_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a),
        "l"(b), "r"(idesc), "r"(acc)
        : "memory");
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
MOEB_DEV void st32(uint32_t addr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        KV_W8(v, 0), KV_W8(v, 8), KV_W8(v, 16), KV_W8(v, 24)
        : "memory");
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
    k.nt = k.ns + max(((pmax + 128) >> 7) - (k.lo >> 7), 0);
    if (pmax < 0) k.ns = k.nt = 0;
    return k;
}
MOEB_DEV int pr_tok(const PrKeys &k, int i) { return (i < k.ns ? i : (k.lo >> 7) + i - k.ns) << 7; }

// natural 8-value word of a row at physical word x of K (the order Q takes too)
template <int FMT, int D>
MOEB_DEV int pr_kword(int x) {
    return FMT == FMT_Q4 ? 8 * ((x >> 1) % (D / 64)) + 2 * (x / (D / 32)) + (x & 1) : 4 * (x % (D / 32)) + x / (D / 32);
}

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

// Largest magnitude (bits) that a row's parameters allow, NaN groups apart; nan: which groups are NaN.
template <int FMT, int NG>
MOEB_DEV uint32_t pr_top(const float (&s)[NG], const float (&b)[NG], unsigned &nan) {
    uint32_t top = 0;
    nan = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const float x = FMT == FMT_Q4 ? fmaxf(fabsf(b[g]), fabsf(fmaf(15.f, s[g], b[g]))) : 6.f * s[g];
        const uint32_t u = __float_as_uint(x);
        if (u < 0x7f800000u && s[g] == s[g]) top = max(top, u);
        else nan |= 1u << g;
    }
    return top;
}

}  // namespace

// part: null, or the workspace of split calls: [splits][T][H][D] sums, then [splits][T][H] (max, sum)
template <int FMT, int D>
__global__ void __launch_bounds__(PT, 1) k_kv_attn_prompt(const KvAttnArgs a, int tiles, float *part) {
    using L = Pr<D>;
    constexpr int NST = L::NST, W4 = D / 32, NG = FMT == FMT_Q4 ? D / 64 : D / 32;
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
            sh.fail = 0;
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
            mbar_init(sh.sfull + i, 1);
            mbar_init(sh.pfull + i, 4);
            mbar_init(sh.ofull + i, 1);
        }
        mbar_fence_init();
        sh.vun = 1.f;
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // ---- queries: fp16 after a power of two per row (the largest value near 2^8), K's order of words, swizzled
    float qmul = 1.f;
    int pos = -1, row_t = 0, row_h = 0;
    if (warp < 8) {
        const int t = warp >> 2, row = (warp & 3) * 32 + lane, R = R0 + t * 128 + row;
        uint4 w[D / 8];
        uint32_t top = 0;
        if (R < NR) {
            const int i = R / a.Gq;
            pos = p0 + i;
            row_t = r0 + i;
            row_h = h * a.Gq + R - i * a.Gq;
            const uint16_t *src = a.q + row_t * a.q_row + row_h * a.q_head;
#pragma unroll
            for (int x = 0; x < D / 8; ++x) w[x] = *reinterpret_cast<const uint4 *>(src + 8 * pr_kword<FMT, D>(x));
        } else {
#pragma unroll
            for (int x = 0; x < D / 8; ++x) w[x] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
            const uint32_t u[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(u[e] & 0x7fffu, (u[e] >> 16) & 0x7fffu));
        }
        const int e = min(max((int)(top >> 7), 9), 254);
        float down = __uint_as_float((uint32_t)(262 - e) << 23);
        qmul = fabsf(a.scale) * __uint_as_float((uint32_t)(e - 8) << 23);
        if (a.scale < 0.f) down = -down;      // the softmax's scale stays positive: it takes the maximum before scaling
        if (a.scale == 0.f) down = 0.f, qmul = 1.f;
        unsigned char *dst = sm + t * L::TILE + row * 128;
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
            const uint32_t u[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
            uint32_t o[4];
#pragma unroll
            for (int e2 = 0; e2 < 4; ++e2) o[e2] = h2(bf16lo(u[e2]) * down, bf16hi(u[e2]) * down);
            *reinterpret_cast<uint4 *>(dst + (x >> 3) * 16384 + (((x & 7) ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        // ------------------------------------------------------------ products of row tile t
        if (warp < 14 && lane == 0 && nk > 0) {
            const int t = warp - 12;
            const uint32_t id_s = (1u << 4) | (16u << 17) | (8u << 24);
            const uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
            const uint32_t ds = tmem + L::S0 + 128 * t, dp = ds + 64, dout = tmem + D * t;
            const uint32_t qa = smem_u32(sm + t * L::TILE);
            bool ok = true;
            for (int j = 0; j < nk; ++j) {
                const int st = j % NST;
                const unsigned ph = (j / NST) & 1;
                if (!pr_wait(sh.kfull + st, ph, &sh.fail)) { ok = false; break; }
                fence_after();
                const uint32_t ka = smem_u32(sm + L::OFF_K + st * L::TILE);
#pragma unroll
                for (int s = 0; s < D / 16; ++s) {
                    const uint32_t off = (s >> 2) * 16384 + (s & 3) * 32;
                    mma_ss(ds, sdesc(qa + off, 16), sdesc(ka + off, 16), id_s, s > 0);
                }
                commit(sh.kempty + st);
                commit(sh.sfull + t);
                if (!pr_wait(sh.vfull + st, ph, &sh.fail) || !pr_wait(sh.pfull + t, j & 1, &sh.fail)) { ok = false; break; }
                fence_after();
                const uint32_t va = smem_u32(sm + L::OFF_V + st * L::TILE);
#pragma unroll
                for (int s = 0; s < 8; ++s) mma_ts(dout, dp + 8 * s, sdesc(va + s * 2048, 16384), id_o, j > 0 || s > 0);
                commit(sh.vempty + st);
            }
            if (!ok) {
                atomicOr(a.c.err, ERR_TIMEOUT);
                *reinterpret_cast<volatile int *>(&sh.fail) = 1;
            }
            commit(sh.ofull + t);
            const int none = 0;
            pr_wait(sh.ofull + t, 0, &none);  // nothing is in flight when TMEM is released
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
        // ------------------------------------------------------------ codes -> fp16 tiles
        const int w = warp - 8, r = lane >> 2, c = lane & 3;
        uint32_t kc[4][W4], vc[4][W4];
        uint32_t kp[4][FMT == FMT_Q4 ? NG : 1], vp[4][FMT == FMT_Q4 ? NG : 1];
        long pid[4];          // of the tile that is fetched next: page, -1: none where one should be, -2: no row sees the key
        unsigned hole_next = 0, hole_now = 0;  // bit per pass: pid == -1
        auto pages = [&](int k) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                pid[i] = -2;
                if (k < k1) {
                    const int j = pr_tok(keys, k) + 32 * i + 8 * w + r;
                    if (j <= pmax && j < Lk && (j >= keys.lo || j < a.sinks)) pid[i] = kv_page(a.c, a.s, b, j);
                }
            }
        };
        auto fetch = [&](int k) {
            hole_next = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (pid[i] == -1) hole_next |= 1u << i;
#pragma unroll
                for (int x = 0; x < W4; ++x) kc[i][x] = vc[i][x] = 0u;
#pragma unroll
                for (int x = 0; x < (FMT == FMT_Q4 ? NG : 1); ++x) kp[i][x] = vp[i][x] = 0u;
                if (pid[i] < 0) continue;
                const size_t row = kv_row(a.c, pid[i], h, pr_tok(keys, k) + 32 * i + 8 * w + r);
                const uint32_t *ks = a.c.kq + row * (D / 8) + c * W4, *vs = a.c.vq + row * (D / 8) + c * W4;
                if (D == 128) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(ks), y = *reinterpret_cast<const uint4 *>(vs);
                    kc[i][0] = x.x; kc[i][1] = x.y; kc[i][W4 - 2] = x.z; kc[i][W4 - 1] = x.w;
                    vc[i][0] = y.x; vc[i][1] = y.y; vc[i][W4 - 2] = y.z; vc[i][W4 - 1] = y.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2 *>(ks), y = *reinterpret_cast<const uint2 *>(vs);
                    kc[i][0] = x.x; kc[i][1] = x.y;
                    vc[i][0] = y.x; vc[i][1] = y.y;
                }
                if (FMT == FMT_Q4) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        kp[i][g] = static_cast<const uint32_t *>(a.c.ks)[row * NG + g];
                        vp[i][g] = static_cast<const uint32_t *>(a.c.vs)[row * NG + g];
                    }
                } else if (D == 128) {
                    kp[i][0] = *reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(a.c.ks) + row * NG);
                    vp[i][0] = *reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(a.c.vs) + row * NG);
                } else {
                    kp[i][0] = *reinterpret_cast<const uint16_t *>(static_cast<const uint8_t *>(a.c.ks) + row * NG);
                    vp[i][0] = *reinterpret_cast<const uint16_t *>(static_cast<const uint8_t *>(a.c.vs) + row * NG);
                }
            }
        };
        // parameters of one row as fp32 (MXFP4: byte 0 of an unseen key stands for 2^-127, times codes of zero)
        auto params = [&](const uint32_t (&p)[FMT == FMT_Q4 ? NG : 1], float (&s)[NG], float (&bb)[NG]) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (FMT == FMT_Q4) {
                    s[g] = bf16lo(p[g]);
                    bb[g] = bf16hi(p[g]);
                } else {
                    s[g] = kv_e8m0((p[0] >> (8 * g)) & 255u);
                    bb[g] = 0.f;
                }
            }
        };
        // the tile's rows, dequantized after multiplication by `mul`; NaN groups of V as zeros
        auto dequant = [&](unsigned char *dst, const uint32_t (&code)[4][W4], const uint32_t (&par)[4][FMT == FMT_Q4 ? NG : 1], float mul,
                           bool isv) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 32 * i + 8 * w + r;
                float s[NG], bb[NG];
                params(par[i], s, bb);
                uint32_t s2[NG], b2[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (isv && !(fabsf(s[g]) <= 3.4028234e38f && fabsf(bb[g]) <= 3.4028234e38f)) s[g] = bb[g] = 0.f;
                    s2[g] = h2(s[g] * mul, s[g] * mul);
                    b2[g] = h2(bb[g] * mul, bb[g] * mul);
                }
#pragma unroll
                for (int x = 0; x < W4; ++x) {
                    // group of physical word c * W4 + x. int4: K (x / 2) of the lane's, V x; MXFP4: K x, V half-words 2 x, 2 x + 1
                    uint4 v;
                    if (FMT == FMT_Q4) {
                        const int g = isv ? x % NG : (x >> 1) % NG;
                        v = pr_word<FMT>(code[i][x], s2[g], b2[g]);
                    } else {
                        const int g = isv ? (2 * x) % NG : x % NG, g1 = isv ? (2 * x + 1) % NG : g;
                        v = pr_word<FMT>(code[i][x], s2[g], s2[g1]);
                    }
                    const int u = c * W4 + x;
                    *reinterpret_cast<uint4 *>(dst + (u >> 3) * 16384 + row * 128 + (((u & 7) ^ (row & 7)) << 4)) = v;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        pages(k0);
        fetch(k0);
        pages(k0 + 1);
        uint32_t vlim = 0;
        float vmul = 1.f, vun = 1.f;
        bool ok = true;
        for (int j = 0; j < nk; ++j) {  // a warp that gave up still comes to the barrier
            const int st = j % NST;
            const unsigned ph = (j / NST + 1) & 1;
            hole_now = hole_next;
            // the tile's largest magnitudes, NaN groups of V
            uint32_t tk = 0, tv = 0;
            unsigned nan[4], any = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float s[NG], bb[NG];
                unsigned drop;
                params(kp[i], s, bb);
                tk = max(tk, pr_top<FMT, NG>(s, bb, drop));
                params(vp[i], s, bb);
                tv = max(tv, pr_top<FMT, NG>(s, bb, nan[i]));
                any |= nan[i];
            }
            tk = __reduce_max_sync(0xffffffffu, tk);
            tv = __reduce_max_sync(0xffffffffu, tv);
            if (lane == 0) {
                sh.mx[j & 1][w][0] = tk;
                sh.mx[j & 1][w][1] = tv;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                tk = max(tk, sh.mx[j & 1][i][0]);
                tv = max(tv, sh.mx[j & 1][i][1]);
            }
            // ---- K
            if (ok && j >= NST && !__all_sync(0xffffffffu, pr_wait(sh.kempty + st, ph, &sh.fail))) ok = false;
            if (ok) {
                const uint32_t e = min(max(tk >> 23, 9u), 254u);
                dequant(sm + L::OFF_K + st * L::TILE, kc, kp, __uint_as_float((262u - e) << 23), false);
                if (w == 0 && lane == 0) sh.kmul[j & 3] = __uint_as_float((e - 8u) << 23);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unsigned x = __ballot_sync(0xffffffffu, (hole_now >> i) & 1u) & 0x11111111u;
                    x = (x | x >> 3) & 0x03030303u;
                    x = (x | x >> 6) & 0x000F000Fu;
                    x = (x | x >> 12) & 0xFFu;
                    if (lane == 0) reinterpret_cast<uint8_t *>(sh.hole[j & 3])[4 * i + w] = (uint8_t)x;
                    if (lane == 0 && x) atomicOr(a.c.err, ERR_PAGE);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(sh.kfull + st);
                // ---- V
                if (j >= NST && !__all_sync(0xffffffffu, pr_wait(sh.vempty + st, ph, &sh.fail))) ok = false;
            }
            if (ok) {
                float fix = 1.f;
                if (tv > vlim) {
                    const uint32_t e = min(max(tv >> 23, 9u), 248u);
                    const float nm = __uint_as_float((262u - e) << 23);
                    fix = nm * vun;
                    vmul = nm;
                    vun = __uint_as_float((e - 8u) << 23);
                    vlim = (e + 6u) << 23;
                }
                dequant(sm + L::OFF_V + st * L::TILE, vc, vp, vmul, true);
                const bool anyw = __any_sync(0xffffffffu, any != 0);
                if (anyw && c == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sh.pm[st][32 * i + 8 * w + r] = (uint8_t)nan[i];
                }
                if (lane == 0) {
                    reinterpret_cast<uint8_t *>(&sh.pz[st])[w] = anyw;
                    if (w == 0) {
                        sh.vfix[st] = fix;
                        sh.vun = vun;
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(sh.vfull + st);
                if (j + 1 < nk) {
                    fetch(k0 + j + 1);
                    pages(k0 + j + 2);
                }
            }
        }
        if (!ok && lane == 0) {
            atomicOr(a.c.err, ERR_TIMEOUT);
            *reinterpret_cast<volatile int *>(&sh.fail) = 1;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
        // ------------------------------------------------------------ softmax of row tile t, a thread per row
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + L::S0 + 128 * t, to = tmem + lanes + D * t;
        const int q0 = R0 + t * 128;
        const int tmin = p0 + q0 / a.Gq, tmax = p0 + (min(q0 + 128, NR) - 1) / a.Gq;  // positions of the tile's rows
        float m = -INFINITY, l = 0.f;
        unsigned poison = 0;
        bool ok = true;
        for (int j = 0; j < nk; ++j) {
            const int st = j % NST, j0 = pr_tok(keys, k0 + j);
            if (!__all_sync(0xffffffffu, pr_wait(sh.sfull + t, j & 1, &sh.fail))) { ok = false; break; }
            fence_after();
            const float sc = fmaxf(qmul * sh.kmul[j & 3], 1.2e-38f);  // above zero: a hidden score of -inf stays -inf
            const unsigned h0 = sh.hole[j & 3][0], h1 = sh.hole[j & 3][1], h2m = sh.hole[j & 3][2], h3 = sh.hole[j & 3][3];
            const bool full = j0 + 127 <= tmin && (!a.window || j0 > tmax - a.window || j0 + 127 < a.sinks) && !(h0 | h1 | h2m | h3);
            const int ce = pos - j0, we = a.window ? pos - a.window + 1 - j0 : -1, se = a.sinks - j0;
            auto mask = [&](float (&v)[64], int half) {
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    const int e = half * 64 + i;
                    const unsigned hw = half ? (i < 32 ? h2m : h3) : (i < 32 ? h0 : h1);
                    const bool vis = e <= ce && (e >= we || e < se) && !((hw >> (i & 31)) & 1u);
                    v[i] = vis ? v[i] : -INFINITY;
                }
            };
            auto top = [&](const float (&v)[64]) {
                float x0 = v[0], x1 = v[1], x2 = v[2], x3 = v[3];
#pragma unroll
                for (int i = 4; i < 64; i += 4) {
                    x0 = fmaxf(x0, v[i]);
                    x1 = fmaxf(x1, v[i + 1]);
                    x2 = fmaxf(x2, v[i + 2]);
                    x3 = fmaxf(x3, v[i + 3]);
                }
                return fmaxf(fmaxf(x0, x1), fmaxf(x2, x3));
            };
            // the row's maximum: keys 0 .. 63, then 64 .. 127, which stay in registers
            float v[64];
            ld32(ts, v);
            ld32(ts + 32, v + 32);
            wait_ld();
            if (!full) mask(v, 0);
            float mt = top(v);
            ld32(ts + 64, v);
            ld32(ts + 96, v + 32);
            wait_ld();
            if (!full) mask(v, 1);
            mt = fmaxf(mt, top(v)) * sc;
            if (!(mt > -INFINITY)) mt = -INFINITY;  // every score a NaN: the weights and the row become NaN
            // V's stage: its power of two, its NaN groups
            if (!__all_sync(0xffffffffu, pr_wait(sh.vfull + st, (j / NST) & 1, &sh.fail))) { ok = false; break; }
            const float vfix = sh.vfix[st];
            if (const unsigned pz = sh.pz[st]) {
                for (int e = 0; e < 128; ++e) {
                    if (!((pz >> (8 * ((e >> 3) & 3))) & 1u)) continue;
                    const unsigned g = sh.pm[st][e];
                    if (g && e <= ce && (e >= we || e < se)) poison |= g;
                }
            }
            // rescale O when a maximum grew far, or V's power of two changed
            float f = 1.f;
            if (mt > m + P_LAZY || (m == -INFINITY && mt > m)) {
                f = m == -INFINITY ? 0.f : ex2p(m - mt);
                m = mt;
                l *= f;
            }
            if (j > 0 && __any_sync(0xffffffffu, f != 1.f || vfix != 1.f)) {
                const float ff = f * vfix;
#pragma unroll
                for (int x = 0; x < D; x += 32) {
                    float o[32];
                    ld32(to + x, o);
                    wait_ld();
                    uint32_t u[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(o[i] * ff);
                    st32(to + x, u);
                }
            }
            const float off = m == -INFINITY ? 0.f : P_OFF - m;
            // weights: keys 64 .. 127 to columns 96 .., then 0 .. 63 to columns 64 .. (S's upper half, both read by then)
            float l0 = 0.f, l1 = 0.f;
            auto weights = [&](const float (&s)[64], uint32_t col) {
                uint32_t u[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float x = ex2p(fmaf(s[2 * i], sc, off)), y = ex2p(fmaf(s[2 * i + 1], sc, off));
                    l0 += x;
                    l1 += y;
                    u[i] = h2(x, y);
                }
                st32(ts + col, u);
            };
            weights(v, 96);
            ld32(ts, v);
            ld32(ts + 32, v + 32);
            wait_ld();
            if (!full) mask(v, 0);
            weights(v, 64);
            wait_st();
            l += l0 + l1;
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sh.pfull + t);
        }
        if (nk > 0 && !__all_sync(0xffffffffu, pr_wait(sh.ofull + t, 0, &sh.fail))) ok = false;
        fence_after();
        if (!ok && lane == 0) {
            atomicOr(a.c.err, ERR_TIMEOUT);
            *reinterpret_cast<volatile int *>(&sh.fail) = 1;
        }
        // ---- the rows' results (m is off by P_OFF against the weights' sum: undone here)
        const float M = m == -INFINITY ? m : m - P_OFF;
        float mul = nk > 0 ? sh.vun : 0.f, Ls = l, sum_m = M;
        const bool have = R0 + t * 128 + (warp & 3) * 32 + lane < NR;
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
        float *pd = part ? part + ((size_t)sp * a.s.T * a.H + orow) * D : nullptr;
#pragma unroll
        for (int x = 0; x < D; x += 32) {
            float o[32];
            if (nk > 0) {
                ld32(to + x, o);
                wait_ld();
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.f;
            }
            if (have) {
            // int4: physical word u of V is word u / G of group u % G; MXFP4: half-word u of 4 values, u / H of group u % H
            constexpr int ST = FMT == FMT_Q4 ? 8 : 4;
#pragma unroll
            for (int i = 0; i < 32; i += ST) {
                const int u = (x + i) / ST, g = u % NG, dim = FMT == FMT_Q4 ? 64 * g + 8 * (u / NG) : 32 * g + 4 * (u / NG);
                float y[ST];
                const bool nanv = (poison >> g) & 1u;
#pragma unroll
                for (int e = 0; e < ST; ++e) y[e] = nanv ? __uint_as_float(0x7fffffffu) : mul == 0.f && l == 0.f ? 0.f : o[i + e] * mul;
                if (part) {
#pragma unroll
                    for (int e = 0; e < ST; e += 4) *reinterpret_cast<float4 *>(pd + dim + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < ST; e += 4)
                        *reinterpret_cast<uint2 *>(a.y + orow * D + dim + e) = make_uint2(pack_bf2(y[e], y[e + 1]), pack_bf2(y[e + 2], y[e + 3]));
                }
            }
            }
            __syncwarp();
        }
        if (have) {
            if (part) reinterpret_cast<float2 *>(part + (size_t)ns * a.s.T * a.H * D)[(size_t)sp * a.s.T * a.H + orow] = make_float2(M, l);
            else if (a.lse) a.lse[orow] = Ls == 0.f ? -INFINITY : (sum_m + log2f(Ls)) * 0.6931471805599453f;
        }
        fence_before();
    }
    __syncthreads();
    if (warp == 12) {
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
