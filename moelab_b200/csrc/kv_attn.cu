// Attention of a few query rows per sequence over the 4-bit cache: decode steps and drafted tokens (layout: kv.cuh).
//
// The rows of a sequence that share a KV head (n tokens x Gq query heads, at most NC = 8 or 16) are the columns of
// one tensor-core tile, so the cache is read once for all of them. The kernel is bound by the cache's bytes when the
// caches are long, and by the chain lengths -> page table -> codes -> sums when they are short.
//
// Work split: the visible keys of every (sequence, KV head) are cut into blocks of 64; all blocks of the call in a row are
// dealt to the CTAs in equal runs, so uneven lengths cost nothing and the host needs to know none of them (a captured
// graph replays with other lengths). A CTA that holds all blocks of a (sequence, head) writes y; otherwise it leaves its
// unnormalised sum, maximum and sum of weights, and k_kv_attn_join joins them.
//
// A warp takes 16 keys of each block, straight from a cp.async ring of its own (no block-wide barrier in the loop), and
// feeds the codes to mma.sync m16n8k16 without dequantizing them:
//   scores^T [16 keys x NC] = K codes . q. int4: 128 + code is one bf16 operation away (code | 0x4300), so with group g's
//     scale s and bias b, score = sum_g s (acc_g - 128 qsum_g) + b qsum_g in fp32. MXFP4: E2M1 codes convert to fp16, q is
//     taken to fp16 with a power of two per row (8 bits of significand fit 11), score = sum_g 2^e acc_g.
//   y^T [D x NC] += V^T codes . P, P = fp16(p * scale of the key's group) after one running power of two per warp, which
//     keeps p * scale in fp16's range whatever the values' size; codes - 8 (int4) or E2M1 in fp16, exact. fp16 and not
//     bf16: P is the only rounding here, 2^-11 keeps it below the result's own 2^-8. int4's bias term is summed in fp32
//     (b + 8 s, so that neither sum is a small difference of large ones).
// Softmax statistics and sums are fp32; a column's maximum is shared by the warp's lanes (three shuffles), warps join at
// the end of a run of blocks. MMA row r is key r / 2 + 4 (r % 2) of its eight, which makes the four keys of a lane's V
// operand consecutive rows of shared memory (no bank conflicts) and costs K nothing.
#include "kv.cuh"

namespace moeb {

namespace {

constexpr int FW = 4, FT = 32 * FW;  // warps per CTA, threads
constexpr int FS = 4;                // ring stages

template <int FMT, int D>
struct Few {
    static constexpr int W = D / 8, G = D / 64, NG = FMT == FMT_Q4 ? D / 64 : D / 32;
    static constexpr int CODE = 16 * D / 2, PAR = FMT == FMT_Q4 ? 16 * G * 4 : 16 * NG;  // bytes of 16 rows
    static constexpr int STAGE = 2 * CODE + 2 * PAR;
};

MOEB_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
MOEB_DEV void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
MOEB_DEV uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// byte i of w: two E2M1 codes (low nibble first) -> f16x2
#define KV_E2M1(B) "{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %1;\n cvt.rn.f16x2.e2m1x2 %0, " B ";\n}"
template <int I>
MOEB_DEV uint32_t e2m1_f16x2(uint32_t w) {
    uint32_t r;
    if (I == 0) asm(KV_E2M1("b0") : "=r"(r) : "r"(w));
    if (I == 1) asm(KV_E2M1("b1") : "=r"(r) : "r"(w));
    if (I == 2) asm(KV_E2M1("b2") : "=r"(r) : "r"(w));
    if (I == 3) asm(KV_E2M1("b3") : "=r"(r) : "r"(w));
    return r;
}
// two E8M0 bytes -> their values (255 is NaN)
MOEB_DEV void e8m0_2(uint32_t two, float &lo, float &hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    lo = bf16lo(r);
    hi = bf16hi(r);
}
MOEB_DEV uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// codes - 8 of nibble P of both halves of t, as f16x2: 1024 + q or 1024 + 16 q by one lop3, then one exact operation
template <int P>
MOEB_DEV uint32_t q4_f16x2(uint32_t t) {
    const uint32_t s = P & 2 ? t >> 8 : t;
    uint32_t r;
    __half2 v;
    if (P & 1) {
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(s), "r"(0x00F000F0u), "r"(0x64006400u));
        v = __hfma2(*reinterpret_cast<__half2 *>(&r), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
    } else {
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(s), "r"(0x000F000Fu), "r"(0x64006400u));
        v = __hadd2(*reinterpret_cast<__half2 *>(&r), __float2half2_rn(-1032.f));
    }
    return *reinterpret_cast<uint32_t *>(&v);
}

// One sequence as the kernels see it: its rows, and the blocks of 64 keys that any of them sees.
struct FewSeq {
    int r0, n, L, lo, ns, nb;
};
// blocks [0, ns): the first tokens; then from lo / 64 on. A sequence with rows has at least one block (its rows are
// written), one with more rows than fit has none.
template <int NC>
MOEB_DEV FewSeq few_seq(const KvAttnArgs &a, int b) {
    FewSeq q;
    int r1;
    kv_rows(a.s, b, q.r0, r1);
    q.n = r1 - q.r0;
    q.L = max(a.s.lens[b], 0);
    const int p0 = max(q.L - q.n, 0);
    q.lo = a.window ? max(p0 - a.window + 1, 0) : 0;
    q.ns = min((min(a.sinks, q.lo) + 63) >> 6, q.lo >> 6);
    q.nb = q.n > 0 && q.n * a.Gq <= NC ? max(q.ns + ((q.L + 63) >> 6) - (q.lo >> 6), 1) : 0;
    return q;
}
MOEB_DEV long few_start(long W, long c, long n) { return W * c / n; }

}  // namespace

// ws: prefix[B + 1] int32 (blocks before each sequence), then 2 partials per CTA: NC rows of D sums, NC (max, sum).
template <int FMT, int D, int NT>
__global__ void __launch_bounds__(FT, NT == 1 ? 4 : 3) k_kv_attn_few(const KvAttnArgs a, int *pre, float *part) {
    using F = Few<FMT, D>;
    constexpr int NC = 8 * NT, NG = F::NG;
    extern __shared__ __align__(16) unsigned char sm[];
    unsigned char *ring = sm + (threadIdx.x >> 5) * (FS * F::STAGE);
    float *so = reinterpret_cast<float *>(sm + FW * FS * F::STAGE);  // [FW][NC][D]
    __shared__ float s_m[FW][NC], s_l[FW][NC];
    __shared__ int s_sum[FW], s_b, s_pre;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
    pdl_wait();

    // every sequence's blocks: prefix sums over the CTA's threads, and the sequence of this CTA's first block
    const int per = (a.s.B + FT - 1) / FT, bb0 = min((int)threadIdx.x * per, a.s.B), bb1 = min(bb0 + per, a.s.B);
    int mine = 0;
    for (int b = bb0; b < bb1; ++b) mine += few_seq<NC>(a, b).nb;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) s_sum[warp] = inc;
    __syncthreads();
    int base = inc - mine, total = 0;
#pragma unroll
    for (int i = 0; i < FW; ++i) {
        if (i < warp) base += s_sum[i];
        total += s_sum[i];
    }
    const long units = (long)total * a.c.Hkv, nct = min((long)gridDim.x, units);
    if (blockIdx.x == 0) {
        int at = base;
        for (int b = bb0; b < bb1; ++b) {
            const FewSeq s = few_seq<NC>(a, b);
            pre[b] = at;
            at += s.nb;
            if (a.only && s.n * a.Gq > NC) atomicOr(a.c.err, ERR_ROWS);
        }
        if (threadIdx.x == 0) pre[a.s.B] = total;
    }
    if ((long)blockIdx.x >= nct) return;
    long u = few_start(units, blockIdx.x, nct);
    const long ue = few_start(units, blockIdx.x + 1, nct), us = u;
    if (u >= (long)base * a.c.Hkv && u < (long)(base + mine) * a.c.Hkv) {
        int at = base, b = bb0;
        for (;; ++b) {
            const int nb = few_seq<NC>(a, b).nb;
            if (u < (long)(at + nb) * a.c.Hkv) break;
            at += nb;
        }
        s_b = b;
        s_pre = at;
    }
    __syncthreads();
    int b = s_b, h;
    FewSeq q = few_seq<NC>(a, b);
    int k0;
    {
        const int off = (int)(u - (long)s_pre * a.c.Hkv);
        h = off / q.nb;
        k0 = off - h * q.nb;
    }
    const int ta = (r >> 1) + 4 * (r & 1);  // this lane's keys of a step: ta and ta + 8

    while (u < ue) {
        // ---- one run of blocks [k0, k1) of (b, h)
        const int k1 = (int)min((long)q.nb, k0 + (ue - u));
        const int p0 = q.L - q.n, plast = q.L - 1;  // positions of the first and the last row
        unsigned ok = 0;
        auto issue = [&](int k) {
            if (k < k1) {
                const int tok = ((k < q.ns ? k : (q.lo >> 6) + k - q.ns) << 6) + 16 * warp;
                const unsigned bit = 1u << (k % FS);
                ok &= ~bit;
                if (tok <= plast && (tok + 15 >= q.lo || tok < a.sinks)) {
                    const long page = kv_page(a.c, a.s, b, tok);
                    if (page < 0) {
                        if (lane == 0) atomicOr(a.c.err, ERR_PAGE);
                    } else {
                        ok |= bit;
                        const size_t row = kv_row(a.c, page, h, tok);
                        unsigned char *st = ring + (k % FS) * F::STAGE;
                        const unsigned char *kq = reinterpret_cast<const unsigned char *>(a.c.kq) + row * (D / 2);
                        const unsigned char *vq = reinterpret_cast<const unsigned char *>(a.c.vq) + row * (D / 2);
#pragma unroll
                        for (int i = 0; i < F::CODE / 512; ++i) {
                            cp_async16(st + (i * 32 + lane) * 16, kq + (i * 32 + lane) * 16);
                            cp_async16(st + F::CODE + (i * 32 + lane) * 16, vq + (i * 32 + lane) * 16);
                        }
                        constexpr int NP = F::PAR / 16;
                        if (lane < 2 * NP) {
                            const unsigned char *ps = static_cast<const unsigned char *>(lane < NP ? a.c.ks : a.c.vs) + row * (F::PAR / 16);
                            cp_async16(st + 2 * F::CODE + lane * 16, ps + (lane % NP) * 16);
                        }
                    }
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < FS - 1; ++i) issue(k0 + i);

        // ---- queries: column nt * 8 + r is row (column / Gq) of the sequence, head h * Gq + column % Gq
        uint32_t qf[NT][D / 16][2];
        float qs[NT][FMT == FMT_Q4 ? NG : 1][2], cs[NT][2];
        int pos[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int col = nt * 8 + r, i = col / a.Gq;
            const bool have = i < q.n;
            const uint16_t *src = a.q + (have ? (q.r0 + i) * a.q_row + (h * a.Gq + col - i * a.Gq) * a.q_head : 0);
            uint4 w[D / 32];
            // words of this lane: int4 2 c, 2 c + 1 of every group of 64; MXFP4 c of every group of 32
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const int word = FMT == FMT_Q4 ? 8 * (j >> 1) + 2 * c + (j & 1) : 4 * j + c;
                w[j] = have ? *reinterpret_cast<const uint4 *>(src + 8 * word) : make_uint4(0, 0, 0, 0);
            }
            float mul = a.scale;
            if (FMT == FMT_FP4) {  // to fp16 by the row's power of two: its largest value near 2^8
                uint32_t t16 = 0;
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const uint32_t ww[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) t16 = max(t16, max(ww[e] & 0x7fffu, (ww[e] >> 16) & 0x7fffu));
                }
                t16 = max(t16, __shfl_xor_sync(0xffffffffu, t16, 1));
                t16 = max(t16, __shfl_xor_sync(0xffffffffu, t16, 2));
                const int e = min(max((int)(t16 >> 7), 9), 254);           // biased exponent of the largest value
                const float down = __uint_as_float((uint32_t)(262 - e) << 23);  // 2^(8 - (e - 127))
                mul = a.scale * __uint_as_float((uint32_t)(e - 8) << 23);
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    uint32_t ww[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) ww[x] = pack_h2(bf16lo(ww[x]) * down, bf16hi(ww[x]) * down);
                    w[j] = make_uint4(ww[0], ww[1], ww[2], ww[3]);
                }
            }
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                qf[nt][2 * j][0] = w[j].x;
                qf[nt][2 * j][1] = w[j].y;
                qf[nt][2 * j + 1][0] = w[j].z;
                qf[nt][2 * j + 1][1] = w[j].w;
            }
            if (FMT == FMT_Q4) {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    float t = 0.f;
#pragma unroll
                    for (int j = 2 * g; j < 2 * g + 2; ++j) {
                        const uint32_t ww[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) t += bf16lo(ww[e]) + bf16hi(ww[e]);
                    }
                    t += __shfl_xor_sync(0xffffffffu, t, 1);
                    t += __shfl_xor_sync(0xffffffffu, t, 2);
                    qs[nt][g][0] = __shfl_sync(0xffffffffu, t, 8 * c);
                    qs[nt][g][1] = __shfl_sync(0xffffffffu, t, 8 * c + 4);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                cs[nt][e] = __shfl_sync(0xffffffffu, mul, 8 * c + 4 * e);
                const int ce = nt * 8 + 2 * c + e, ie = ce / a.Gq;
                pos[nt][e] = ie < q.n ? p0 + ie : -1;  // a column without a row sees nothing
            }
        }

        float o[NT][D / 16][4], m[NT][2], l[NT][2], bs[NT][FMT == FMT_Q4 ? NG : 1][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[nt][e] = -INFINITY;
                l[nt][e] = 0.f;
#pragma unroll
                for (int g = 0; g < (FMT == FMT_Q4 ? NG : 1); ++g) bs[nt][g][e] = 0.f;
            }
        }
        uint32_t vlim = 0;           // bits of the largest value scale that the running power of two takes
        float vmul = 1.f, vun = 1.f;  // that power and its inverse

        for (int k = k0; k < k1; ++k) {
            cp_wait<FS - 2>();
            __syncwarp();
            if (ok >> (k % FS) & 1) {
                const unsigned char *st = ring + (k % FS) * F::STAGE;
                const int tok = ((k < q.ns ? k : (q.lo >> 6) + k - q.ns) << 6) + 16 * warp;
                // ---- scores of keys ta, ta + 8 for columns 2 c, 2 c + 1
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
                uint32_t wa[D / 32], wb[D / 32];
                {
                    const unsigned char *ra = st + ta * (D / 2) + c * (D / 8);
                    if (D == 128) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(ra), y = *reinterpret_cast<const uint4 *>(ra + 4 * D);
                        wa[0] = x.x; wa[1] = x.y; wa[D / 32 - 2] = x.z; wa[D / 32 - 1] = x.w;
                        wb[0] = y.x; wb[1] = y.y; wb[D / 32 - 2] = y.z; wb[D / 32 - 1] = y.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2 *>(ra), y = *reinterpret_cast<const uint2 *>(ra + 4 * D);
                        wa[0] = x.x; wa[1] = x.y;
                        wb[0] = y.x; wb[1] = y.y;
                    }
                }
                const unsigned char *pk = st + 2 * F::CODE, *pv = pk + F::PAR;
                if (FMT == FMT_Q4) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        float acc[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t ua = wa[(x >> 1) * NG + g], ub = wb[(x >> 1) * NG + g];
                            const int p = 2 * (x & 1);
                            const uint32_t A[4] = {q4pair(ua, p), q4pair(ub, p), q4pair(ua, p + 1), q4pair(ub, p + 1)};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_bf16(acc[nt], A, qf[nt][4 * g + x][0], qf[nt][4 * g + x][1]);
                        }
                        const uint32_t sa = *reinterpret_cast<const uint32_t *>(pk + (ta * NG + g) * 4);
                        const uint32_t sb = *reinterpret_cast<const uint32_t *>(pk + ((ta + 8) * NG + g) * 4);
                        const float xa = bf16lo(sa), ya = fmaf(-128.f, xa, bf16hi(sa)), xb = bf16lo(sb), yb = fmaf(-128.f, xb, bf16hi(sb));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                s[nt][e] += fmaf(xa, acc[nt][e], ya * qs[nt][g][e]);
                                s[nt][2 + e] += fmaf(xb, acc[nt][2 + e], yb * qs[nt][g][e]);
                            }
                        }
                    }
                } else {
                    float xa[NG], xb[NG];
#pragma unroll
                    for (int g = 0; g < NG; g += 2) {
                        e8m0_2(*reinterpret_cast<const uint16_t *>(pk + ta * NG + g), xa[g], xa[g + 1]);
                        e8m0_2(*reinterpret_cast<const uint16_t *>(pk + (ta + 8) * NG + g), xb[g], xb[g + 1]);
                    }
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        float acc[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
                        // half-words 2 c (product 0) and 2 c + 1 of the group
                        const int x0 = g >> 1, x1 = NG / 2 + (g >> 1);
                        uint32_t A0[4], A1[4];
                        if (g & 1) {
                            A0[0] = e2m1_f16x2<2>(wa[x0]); A0[1] = e2m1_f16x2<2>(wb[x0]); A0[2] = e2m1_f16x2<3>(wa[x0]); A0[3] = e2m1_f16x2<3>(wb[x0]);
                            A1[0] = e2m1_f16x2<2>(wa[x1]); A1[1] = e2m1_f16x2<2>(wb[x1]); A1[2] = e2m1_f16x2<3>(wa[x1]); A1[3] = e2m1_f16x2<3>(wb[x1]);
                        } else {
                            A0[0] = e2m1_f16x2<0>(wa[x0]); A0[1] = e2m1_f16x2<0>(wb[x0]); A0[2] = e2m1_f16x2<1>(wa[x0]); A0[3] = e2m1_f16x2<1>(wb[x0]);
                            A1[0] = e2m1_f16x2<0>(wa[x1]); A1[1] = e2m1_f16x2<0>(wb[x1]); A1[2] = e2m1_f16x2<1>(wa[x1]); A1[3] = e2m1_f16x2<1>(wb[x1]);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_f16(acc[nt], A0, qf[nt][2 * g][0], qf[nt][2 * g][1]);
                            mma_f16(acc[nt], A1, qf[nt][2 * g + 1][0], qf[nt][2 * g + 1][1]);
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                s[nt][e] = fmaf(xa[g], acc[nt][e], s[nt][e]);
                                s[nt][2 + e] = fmaf(xb[g], acc[nt][2 + e], s[nt][2 + e]);
                            }
                        }
                    }
                }
                // ---- the value scales of keys ta, ta + 8 (zero where no row sees the key: what lies there is not looked at)
                float va[NG], vb[NG], ba[NG], bb[NG];
                const int ja = tok + ta, jb = ja + 8;
                const bool full = tok + 15 <= p0 && (!a.window || tok > plast - a.window || tok + 15 < a.sinks);
                if (FMT == FMT_Q4) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const uint32_t sa = *reinterpret_cast<const uint32_t *>(pv + (ta * NG + g) * 4);
                        const uint32_t sb = *reinterpret_cast<const uint32_t *>(pv + ((ta + 8) * NG + g) * 4);
                        va[g] = bf16lo(sa);
                        ba[g] = fmaf(8.f, va[g], bf16hi(sa));
                        vb[g] = bf16lo(sb);
                        bb[g] = fmaf(8.f, vb[g], bf16hi(sb));
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < NG; g += 2) {
                        e8m0_2(*reinterpret_cast<const uint16_t *>(pv + ta * NG + g), va[g], va[g + 1]);
                        e8m0_2(*reinterpret_cast<const uint16_t *>(pv + (ta + 8) * NG + g), vb[g], vb[g + 1]);
                    }
                }
                if (!full) {
                    const bool sa = ja <= plast && (ja >= q.lo || ja < a.sinks), sb = jb <= plast && (jb >= q.lo || jb < a.sinks);
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        va[g] = sa ? va[g] : 0.f;
                        vb[g] = sb ? vb[g] : 0.f;
                        if (FMT == FMT_Q4) {
                            ba[g] = sa ? ba[g] : 0.f;
                            bb[g] = sb ? bb[g] : 0.f;
                        }
                    }
                }
                uint32_t top = 0;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t x = __float_as_uint(va[g]) & 0x7fffffffu, y = __float_as_uint(vb[g]) & 0x7fffffffu;
                    top = max(top, max(x < 0x7f800000u ? x : 0u, y < 0x7f800000u ? y : 0u));
                }
                top = __reduce_max_sync(0xffffffffu, top);
                float fix = 1.f;
                if (top > vlim) {  // larger than the power of two takes: scale to 2^8, with room to 2^14
                    const uint32_t e = min(max(top >> 23, 9u), 248u);
                    const float nm = __uint_as_float((262u - e) << 23);
                    fix = nm * vun;
                    vmul = nm;
                    vun = __uint_as_float((e - 8u) << 23);
                    vlim = (e + 6u) << 23;
                }
                // ---- mask, running maximum, weights
                bool grew = fix != 1.f;
                float f[NT][2];
                bool vis[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s[nt][e] *= cs[nt][e];
                        s[nt][2 + e] *= cs[nt][e];
                        vis[nt][e] = vis[nt][2 + e] = true;
                        if (!full) {
                            const int p = pos[nt][e];
                            vis[nt][e] = ja <= p && (!a.window || ja > p - a.window || ja < a.sinks);
                            vis[nt][2 + e] = jb <= p && (!a.window || jb > p - a.window || jb < a.sinks);
                            if (!vis[nt][e]) s[nt][e] = -INFINITY;
                            if (!vis[nt][2 + e]) s[nt][2 + e] = -INFINITY;
                        }
                        float t = fmaxf(s[nt][e], s[nt][2 + e]);
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                        const float mn = fmaxf(m[nt][e], t);
                        grew |= mn > m[nt][e];
                        const float use = mn == -INFINITY ? 0.f : mn;
                        f[nt][e] = ex2(m[nt][e] - use);
                        m[nt][e] = mn;
                        s[nt][e] = ex2(s[nt][e] - use);
                        s[nt][2 + e] = ex2(s[nt][2 + e] - use);
                    }
                }
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            l[nt][e] *= f[nt][e];
                            if (FMT == FMT_Q4) {
#pragma unroll
                                for (int g = 0; g < NG; ++g) bs[nt][g][e] *= f[nt][e];
                            }
                            const float ff = f[nt][e] * fix;
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) {
                                o[nt][i][e] *= ff;
                                o[nt][i][2 + e] *= ff;
                            }
                        }
                    }
                }
                uint32_t pf[NT][NG][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) l[nt][e] += s[nt][e] + s[nt][2 + e];
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const float xa = va[g] * vmul, xb = vb[g] * vmul;
                        float w[4] = {s[nt][0] * xa, s[nt][1] * xa, s[nt][2] * xb, s[nt][3] * xb};
                        if (!full) {  // a key that one row sees and another does not may hold a NaN
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] = vis[nt][e] ? w[e] : 0.f;
                        }
                        pf[nt][g][0] = transpose8(pack_h2(w[0], w[1]));
                        pf[nt][g][1] = transpose8(pack_h2(w[2], w[3]));
                        if (FMT == FMT_Q4) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float x = s[nt][e] * ba[g], y = s[nt][2 + e] * bb[g];
                                bs[nt][g][e] += (vis[nt][e] ? x : 0.f) + (vis[nt][2 + e] ? y : 0.f);
                            }
                        }
                    }
                }
                // ---- values: keys c, c + 4, c + 8, c + 12
                const unsigned char *rv = st + F::CODE + c * (D / 2) + r * (D / 16);
                uint32_t vw[4][D / 64];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if (D == 128) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(rv + t * 2 * D);
                        vw[t][0] = x.x;
                        vw[t][D / 64 - 1] = x.y;
                    } else {
                        vw[t][0] = *reinterpret_cast<const uint32_t *>(rv + t * 2 * D);
                    }
                }
#pragma unroll
                for (int g = 0; g < D / 64; ++g) {
                    if (FMT == FMT_Q4) {
                        const uint32_t l0 = __byte_perm(vw[0][g], vw[1][g], 0x5410), h0 = __byte_perm(vw[0][g], vw[1][g], 0x7632);
                        const uint32_t l1 = __byte_perm(vw[2][g], vw[3][g], 0x5410), h1 = __byte_perm(vw[2][g], vw[3][g], 0x7632);
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            uint32_t A[4];
                            if (p == 0) { A[0] = q4_f16x2<0>(l0); A[1] = q4_f16x2<0>(h0); A[2] = q4_f16x2<0>(l1); A[3] = q4_f16x2<0>(h1); }
                            if (p == 1) { A[0] = q4_f16x2<1>(l0); A[1] = q4_f16x2<1>(h0); A[2] = q4_f16x2<1>(l1); A[3] = q4_f16x2<1>(h1); }
                            if (p == 2) { A[0] = q4_f16x2<2>(l0); A[1] = q4_f16x2<2>(h0); A[2] = q4_f16x2<2>(l1); A[3] = q4_f16x2<2>(h1); }
                            if (p == 3) { A[0] = q4_f16x2<3>(l0); A[1] = q4_f16x2<3>(h0); A[2] = q4_f16x2<3>(l1); A[3] = q4_f16x2<3>(h1); }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][4 * g + p], A, pf[nt][g][0], pf[nt][g][1]);
                        }
                    } else {
                        const uint32_t mk = 0x0F0F0F0Fu;
                        const uint32_t e0 = (vw[0][g] & mk) | ((vw[1][g] << 4) & ~mk), d0 = ((vw[0][g] >> 4) & mk) | (vw[1][g] & ~mk);
                        const uint32_t e1 = (vw[2][g] & mk) | ((vw[3][g] << 4) & ~mk), d1 = ((vw[2][g] >> 4) & mk) | (vw[3][g] & ~mk);
                        const uint32_t A0[4] = {e2m1_f16x2<0>(e0), e2m1_f16x2<0>(d0), e2m1_f16x2<0>(e1), e2m1_f16x2<0>(d1)};
                        const uint32_t A1[4] = {e2m1_f16x2<1>(e0), e2m1_f16x2<1>(d0), e2m1_f16x2<1>(e1), e2m1_f16x2<1>(d1)};
                        const uint32_t A2[4] = {e2m1_f16x2<2>(e0), e2m1_f16x2<2>(d0), e2m1_f16x2<2>(e1), e2m1_f16x2<2>(d1)};
                        const uint32_t A3[4] = {e2m1_f16x2<3>(e0), e2m1_f16x2<3>(d0), e2m1_f16x2<3>(e1), e2m1_f16x2<3>(d1)};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_f16(o[nt][4 * g + 0], A0, pf[nt][2 * g][0], pf[nt][2 * g][1]);
                            mma_f16(o[nt][4 * g + 1], A1, pf[nt][2 * g][0], pf[nt][2 * g][1]);
                            mma_f16(o[nt][4 * g + 2], A2, pf[nt][2 * g + 1][0], pf[nt][2 * g + 1][1]);
                            mma_f16(o[nt][4 * g + 3], A3, pf[nt][2 * g + 1][0], pf[nt][2 * g + 1][1]);
                        }
                    }
                }
            }
            __syncwarp();
            issue(k + FS - 1);
        }
        cp_wait<0>();

        // ---- the warps' sums join in shared memory
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int x = 4; x <= 16; x <<= 1) {
                    l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
                    if (FMT == FMT_Q4) {
#pragma unroll
                        for (int g = 0; g < NG; ++g) bs[nt][g][e] += __shfl_xor_sync(0xffffffffu, bs[nt][g][e], x);
                    }
                }
                if (r == 0) {
                    s_m[warp][nt * 8 + 2 * c + e] = m[nt][e];
                    s_l[warp][nt * 8 + 2 * c + e] = l[nt][e];
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = nt * 8 + 2 * c + e;
                float M = s_m[0][col];
#pragma unroll
                for (int i = 1; i < FW; ++i) M = fmaxf(M, s_m[i][col]);
                const float fm = ex2(m[nt][e] - (M == -INFINITY ? 0.f : M));
                float *dst = so + (warp * NC + col) * D;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    // int4: tile 4 g + p is elements 2 p, 2 p + 1 of words r of group g; MXFP4: tile 2 g + x is elements
                    // 4 r + 2 x, 4 r + 2 x + 1 of group g (of 32)
                    const int dim = FMT == FMT_Q4 ? 64 * (i >> 2) + 8 * r + 2 * (i & 3) : 32 * (i >> 1) + 4 * r + 2 * (i & 1);
                    const float add = FMT == FMT_Q4 ? bs[nt][i >> 2 < NG ? i >> 2 : 0][e] : 0.f;
                    float2 v;
                    v.x = fmaf(o[nt][i][e], vun, add) * fm;
                    v.y = fmaf(o[nt][i][2 + e], vun, add) * fm;
                    *reinterpret_cast<float2 *>(dst + dim) = v;
                }
            }
        }
        __syncthreads();
        const bool whole = k0 == 0 && k1 == q.nb;
        float *pt = part + ((size_t)blockIdx.x * 2 + (u == us ? 0 : 1)) * (NC * (D + 2));
        for (int i = threadIdx.x; i < q.n * a.Gq * (D / 4); i += FT) {
            const int col = i / (D / 4), d4 = i % (D / 4);
            float M = s_m[0][col], L = 0.f;
#pragma unroll
            for (int x = 1; x < FW; ++x) M = fmaxf(M, s_m[x][col]);
            const float use = M == -INFINITY ? 0.f : M;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < FW; ++x) {
                const float4 w = *reinterpret_cast<const float4 *>(so + (x * NC + col) * D + 4 * d4);
                v.x += w.x;
                v.y += w.y;
                v.z += w.z;
                v.w += w.w;
                L += s_l[x][col] * ex2(s_m[x][col] - use);
            }
            if (whole) {
                const int ri = col / a.Gq, head = h * a.Gq + col - ri * a.Gq;
                kv_finish<D>(a, q.r0 + ri, head, d4, v, M, L);
            } else {
                *reinterpret_cast<float4 *>(pt + col * D + 4 * d4) = v;
                if (d4 == 0) *reinterpret_cast<float2 *>(pt + NC * D + 2 * col) = make_float2(M, L);
            }
        }
        __syncthreads();

        // ---- the next run
        u += k1 - k0;
        k0 = 0;
        if (u < ue && ++h == a.c.Hkv) {
            h = 0;
            do q = few_seq<NC>(a, ++b);
            while (q.nb == 0);
        }
    }
}

// Joins the partial sums of every (sequence, KV head) whose blocks more than one CTA had: one CTA per column, its warps
// share the partials.
template <int D, int NT>
__global__ void __launch_bounds__(256) k_kv_attn_join(const KvAttnArgs a, const int *pre, const float *part, int grid) {
    constexpr int NC = 8 * NT;
    __shared__ float s_m[8], s_l[8];
    __shared__ float so[8][D];
    pdl_wait();
    const int col = blockIdx.y, h = blockIdx.x % a.c.Hkv, b = blockIdx.x / a.c.Hkv;
    const int at = pre[b], nb = pre[b + 1] - at;
    if (nb < 2) return;  // none, or one block: one CTA had it
    const FewSeq q = few_seq<NC>(a, b);
    if (col >= q.n * a.Gq) return;
    const long units = (long)pre[a.s.B] * a.c.Hkv, n = min((long)grid, units);
    const long u0 = (long)at * a.c.Hkv + (long)h * nb, u1 = u0 + nb;
    const int c0 = (int)(((u0 + 1) * n - 1) / units), c1 = (int)((u1 * n - 1) / units);  // CTAs of the first and last block
    if (c0 == c1) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int E = D / 32;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
    for (int x = c0 + warp; x <= c1; x += 8) {
        const float *pt = part + ((size_t)x * 2 + (few_start(units, x, n) >= u0 ? 0 : 1)) * (NC * (D + 2));
        const float2 ml = *reinterpret_cast<const float2 *>(pt + NC * D + 2 * col);
        const float mn = fmaxf(m, ml.x), use = mn == -INFINITY ? 0.f : mn;
        const float f = ex2(m - use), g = ex2(ml.x - use);
        m = mn;
        l = l * f + ml.y * g;
        const float *src = pt + col * D + lane * E;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = o[i] * f + src[i] * g;
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) so[warp][lane * E + i] = o[i];
    __syncthreads();
    if (threadIdx.x >= D / 4) return;
    float M = s_m[0], L = 0.f;
#pragma unroll
    for (int i = 1; i < 8; ++i) M = fmaxf(M, s_m[i]);
    const float use = M == -INFINITY ? 0.f : M;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = ex2(s_m[i] - use);
        const float4 w = *reinterpret_cast<const float4 *>(&so[i][4 * threadIdx.x]);
        v.x += w.x * f;
        v.y += w.y * f;
        v.z += w.z * f;
        v.w += w.w * f;
        L += s_l[i] * f;
    }
    const int ri = col / a.Gq;
    kv_finish<D>(a, q.r0 + ri, h * a.Gq + col - ri * a.Gq, threadIdx.x, v, M, L);
}

template <int FMT, int D, int NT>
size_t kv_few_smem() {
    return (size_t)FW * FS * Few<FMT, D>::STAGE + (size_t)FW * 8 * NT * D * 4;
}

#define KV_INST(F, D, NT)                                                          \
    template __global__ void k_kv_attn_few<F, D, NT>(const KvAttnArgs, int *, float *); \
    template size_t kv_few_smem<F, D, NT>();
KV_INST(FMT_Q4, 64, 1)
KV_INST(FMT_Q4, 128, 1)
KV_INST(FMT_FP4, 64, 1)
KV_INST(FMT_FP4, 128, 1)
KV_INST(FMT_Q4, 64, 2)
KV_INST(FMT_Q4, 128, 2)
KV_INST(FMT_FP4, 64, 2)
KV_INST(FMT_FP4, 128, 2)
template __global__ void k_kv_attn_join<64, 1>(const KvAttnArgs, const int *, const float *, int);
template __global__ void k_kv_attn_join<64, 2>(const KvAttnArgs, const int *, const float *, int);
template __global__ void k_kv_attn_join<128, 1>(const KvAttnArgs, const int *, const float *, int);
template __global__ void k_kv_attn_join<128, 2>(const KvAttnArgs, const int *, const float *, int);

}  // namespace moeb
