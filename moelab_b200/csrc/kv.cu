// Writing K and V rows into the 4-bit cache, and reading them back (layout: kv.cuh). Both are one pass over memory: per value
// two bytes of bf16 and 0.56 (int4) or 0.53 (MXFP4) of the cache. A thread has what one lane of the cache's readers has: the
// same word of every group of a row (int4: 1 / 8 of the row, MXFP4: 1 / 4; rows of 64 values: of K's and V's), so that its codes
// are one load or store and the page arithmetic is done once for all of them; and KV_U tokens of one head, so that as many loads
// are in flight (one token in calls too small to fill the GPU). The lanes of a group reduce its extremes by shuffles.
// Measured with 65,536 tokens of 1,024 values each of K and V (8 heads of 128 / 16 of 64), copies of the same bytes at 6.56
// TB/s being 52 us:
//   write  int4 72 / 75 us (4.8 / 4.6 TB/s; bound by instructions), MXFP4 55 / 62 us (6.2 / 5.5 TB/s)
//   read   int4 62 / 70 us (5.5 / 4.9 TB/s), MXFP4 61 / 67 us (5.6 / 5.1 TB/s)
// A call of one token is bound by its launch: written and read back, 4.7 us in a graph.
#include "kv.cuh"

namespace moeb {

constexpr int KV_U = 4;
template <int FMT, int D>
struct Wd {
    static constexpr int LR = FMT == FMT_Q4 ? 8 : 4;  // lanes per row, = words of 8 values in a group
    static constexpr int NG = D / (8 * LR);           // groups in a row, = words per lane
    static constexpr int A = KV_BOTH(D) ? 2 : 1;      // arrays that a thread has rows of: K or V, or both
    static constexpr int NW = NG * A;                 // its words
    static constexpr int R = 128 / LR;                // rows per CTA and pass
};
template <int N>
struct Vec { using T = uint32_t; };
template <>
struct Vec<2> { using T = uint2; };
template <>
struct Vec<4> { using T = uint4; };
// physical codes of a lane <-> its words (values 8 (LR g + w) .. of group g): int4 as they are; MXFP4 two half-words apart
template <int FMT, int N>
MOEB_DEV void lane_words(const uint32_t (&in)[N], uint32_t (&out)[N], bool to_words) {
#pragma unroll
    for (int g = 0; g < N; ++g) {
        if (FMT == FMT_Q4) out[g] = in[g];
        else if (to_words) out[g] = __byte_perm(in[g / 2], in[N / 2 + g / 2], g & 1 ? 0x7632 : 0x5410);
        else out[g] = g < N / 2 ? __byte_perm(in[2 * g], in[2 * g + 1], 0x5410) : __byte_perm(in[2 * g - N], in[2 * g + 1 - N], 0x7632);
    }
}

// int4: a group's 64 values lie in 8 neighbouring lanes, 8 in each. The operations are those of the weight quantizer
// (quant.cu), so a cache row equals mx.quantize of it. A group that holds an infinity or a NaN, or whose span passes fp32, is
// stored with NaN parameters: it reads back as NaN everywhere, and nothing else is touched by it. Bound by its instructions, not
// by memory: pairs of values go through packed operations, and each of the eight lanes works out the parameters of one of the
// eight groups that they have in four tokens (all lanes those of every group: 84 against 72 us).
struct Q4Group {
    float scale, bias, inv;  // inv = 0: all codes are 0
    uint32_t par;            // as stored; 0: all zeros
};
// (largest, -smallest) of the group; a NaN stays
MOEB_DEV __nv_bfloat162 kv_q4_range(const uint4 u) {
    const __nv_bfloat162 x0 = *reinterpret_cast<const __nv_bfloat162 *>(&u.x), x1 = *reinterpret_cast<const __nv_bfloat162 *>(&u.y),
                         x2 = *reinterpret_cast<const __nv_bfloat162 *>(&u.z), x3 = *reinterpret_cast<const __nv_bfloat162 *>(&u.w);
    const __nv_bfloat162 mx = __hmax2_nan(__hmax2_nan(x0, x1), __hmax2_nan(x2, x3)), mn = __hmin2_nan(__hmin2_nan(x0, x1), __hmin2_nan(x2, x3));
    __nv_bfloat162 m = __halves2bfloat162(__hmax_nan(__low2bfloat16(mx), __high2bfloat16(mx)), __hneg(__hmin_nan(__low2bfloat16(mn), __high2bfloat16(mn))));
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) m = __hmax2_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
MOEB_DEV Q4Group kv_q4_group(const __nv_bfloat162 m) {
    Q4Group g;
    const float hi = __low2float(m), lo = -__high2float(m);
    const bool mask = fabsf(lo) > fabsf(hi);
    float scale = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
    const bool bad = !(scale <= 3.4028234e38f);  // NaN, infinity, or a span that is none
    scale = scale > 1e-7f ? scale : 1e-7f;
    scale = mask ? scale : -scale;
    const float edge = mask ? lo : hi;
    const float q0 = rintf(__fdiv_rn(edge, scale));
    g.bias = 0.0f;
    if (q0 != 0.0f) {
        scale = __fdiv_rn(edge, q0);
        g.bias = edge;
    }
    g.scale = scale;
    // q0 = 0: the largest magnitude is below half the smallest scale, every code is 0 and the values are zeros. The weight
    // quantizer keeps that scale; here it is 0, so that attention, which goes by the parameters where it weighs values' sizes
    // against one another, meets no scale of 2^-23 that belongs to nothing.
    g.par = bad ? 0x7fff7fffu : q0 == 0.0f ? 0u : (uint32_t)f2bf(scale) | ((uint32_t)f2bf(g.bias) << 16);
    g.inv = bad || q0 == 0.0f ? 0.0f : __frcp_rn(scale);
    return g;
}
MOEB_DEV uint32_t kv_quant_q4(const uint4 u, const Q4Group &g) {
    const float scale = g.scale, bias = g.bias, inv = g.inv;
    // code = rint(d / scale), d = v - bias, the quotient rounded to fp32; it is not negative, as the bias is the end of the
    // range that the scale's sign points away from. Quotient: q = d * (1 / scale), then q + (d - q * scale) * (1 / scale) with the
    // difference exact in a fused product, which is the quotient's rounding when 1 / scale is rounded to nearest (P. Markstein,
    // Computation of elementary functions on the IBM RISC System/6000, 1990). No branch: bf16 values fall on halves so often
    // that half of the warps took one that divided only there.
    // Adding 1.5 * 2^23 rounds to a whole number, to even as rintf does, and leaves it in the low bits.
    const uint64_t b2 = pair(-bias, -bias), i2 = pair(inv, inv), s2 = pair(-scale, -scale), up = pair(12582912.f, 12582912.f);
    const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t d = add2(pair(bf16lo(uu[i]), bf16hi(uu[i])), b2), r = mul2(d, i2);
        const uint64_t q = add2(fma2(fma2(r, s2, d), i2, r), up);
        // value 2 i's code in the low half, 2 i + 1's in the high one: nibbles i and i + 4 of the word
        word += __vminu2(__byte_perm((uint32_t)q, (uint32_t)(q >> 32), 0x5410), 0x000f000fu) << (4 * i);
    }
    return inv == 0.f ? 0u : word;
}
MOEB_DEV uint32_t kv_quant_fp4(const uint4 u, uint32_t &par) {
    const float v[8] = {bf16lo(u.x), bf16hi(u.x), bf16lo(u.y), bf16hi(u.y), bf16lo(u.z), bf16hi(u.z), bf16lo(u.w), bf16hi(u.w)};
    uint32_t top = 0;  // the largest magnitude's bits: they order as the values do, with NaN on top
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    if (top >= 0x7f800000u) {
        par = 255u;
        return 0u;
    }
    // exponent of the largest value less that of E2M1's largest (4 .. 6 = 2^2); bf16 subnormals give the lowest byte
    const int e = max((int)(top >> 23) - 127 - 2, -127);
    par = (uint32_t)(e + 127);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);  // 2^-e, e <= 125
    // to the nearest E2M1 value, halves to the even code, 6 at most, the sign kept
    uint32_t word;
    asm("{\n .reg .b8 b0, b1, b2, b3;\n cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n mov.b32 %0, {b0, b1, b2, b3};\n}"
        : "=r"(word)
        : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv), "f"(v[6] * inv), "f"(v[7] * inv));
    return word;
}

// CTA: R * passes tokens of one head, K or V (blockIdx.y = 2 * head + is V) or both (blockIdx.y = head)
template <int FMT, int D>
__global__ void __launch_bounds__(128) k_kv_write(const KvWriteArgs a) {
    using X = Wd<FMT, D>;
    constexpr int NG = X::NG, A = X::A, NW = X::NW;
    const int w = threadIdx.x % X::LR, h = A == 2 ? blockIdx.y : blockIdx.y >> 1;
    const bool isv = A == 1 && (blockIdx.y & 1);
    const uint16_t *src[A];
    long stride[A];
    uint32_t *codes[A];
    unsigned char *ps[A];
#pragma unroll
    for (int x = 0; x < A; ++x) {
        const bool v = isv || x == 1;
        src[x] = (v ? a.v + h * a.v_head : a.k + h * a.k_head) + 8 * w;
        stride[x] = v ? a.v_row : a.k_row;
        codes[x] = (v ? a.c.vq : a.c.kq) + w * NG;
        ps[x] = static_cast<unsigned char *>(v ? a.c.vs : a.c.ks);
    }
    const int t0 = (int)blockIdx.x * (X::R * a.passes) + (int)threadIdx.x / X::LR;
    pdl_wait();
    auto fetch = [&](int t, bool any, uint4 (&u)[NW]) {
#pragma unroll
        for (int g = 0; g < NW; ++g)
            u[g] = any && t < a.s.T ? *reinterpret_cast<const uint4 *>(src[g / NG] + t * stride[g / NG] + g % NG * (8 * X::LR)) : make_uint4(0, 0, 0, 0);
    };
    constexpr int U = FMT == FMT_Q4 ? KV_U : 1;
    uint4 next[U][NW];
#pragma unroll
    for (int i = 0; i < U; ++i) fetch(t0 + i * X::R, i < a.passes, next[i]);
    // where the rows of the warp's passes go, a lane per row: its position, its page (-1: nowhere)
    constexpr int WR = 32 / X::LR;  // a warp's rows in a pass
    const int lane = threadIdx.x & 31;
    int at = -1, to = -1;
    {
        const int t = t0 - lane / X::LR + lane / WR * X::R + lane % WR;
        if (lane / WR < a.passes && t < a.s.T) {
            int r0, r1;
            const int b = kv_seq_of(a.s, t, r0, r1);
            if (b >= 0) at = a.s.lens[b] - (r1 - t);
            if (at >= 0) {
                to = (int)kv_page(a.c, a.s, b, at);
                if (to < 0 && blockIdx.y == 0) atomicOr(a.c.err, ERR_PAGE);
            }
        }
        __syncwarp();
    }
    using T = typename Vec<NG>::T;
    auto store = [&](int i, const uint32_t (&word)[NW], const uint32_t *par) {
        const int page = __shfl_sync(0xffffffffu, to, i * WR + lane / X::LR), p = __shfl_sync(0xffffffffu, at, i * WR + lane / X::LR);
        if (page < 0) return;
        const size_t row = kv_row(a.c, page, h, p);
#pragma unroll
        for (int x = 0; x < A; ++x) {
            uint32_t in[NG], out[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) in[g] = word[x * NG + g];
            lane_words<FMT>(in, out, false);
            *reinterpret_cast<T *>(codes[x] + row * (D / 8)) = *reinterpret_cast<const T *>(out);
            if (FMT != FMT_Q4 && w == 0) {
                const uint32_t *e = par + x * NG;
                if (NG == 4) *reinterpret_cast<uint32_t *>(ps[x] + row * NG) = e[0] | e[1] << 8 | e[NG - 2] << 16 | e[NG - 1] << 24;
                else *reinterpret_cast<uint16_t *>(ps[x] + row * NG) = (uint16_t)(e[0] | e[1 % NG] << 8);
            }
        }
    };
    // every lane takes part in the shuffles; a group's lanes are all inside one row
    if constexpr (FMT == FMT_Q4) {
        static_assert(KV_U * NW == X::LR, "a lane per group of a row's passes");
        __nv_bfloat162 m;
#pragma unroll
        for (int i = 0; i < KV_U; ++i) {
            if (i >= a.passes) break;
#pragma unroll
            for (int g = 0; g < NW; ++g) {
                const __nv_bfloat162 x = kv_q4_range(next[i][g]);
                if (i * NW + g == 0 || w == i * NW + g) m = x;
            }
        }
        const Q4Group mine = kv_q4_group(m);
#pragma unroll
        for (int i = 0; i < KV_U; ++i) {
            if (i >= a.passes) break;
            uint32_t word[NW];
#pragma unroll
            for (int g = 0; g < NW; ++g) {
                const int from = ((int)threadIdx.x & 24) | (i * NW + g);
                Q4Group q;
                q.scale = __shfl_sync(0xffffffffu, mine.scale, from);
                q.bias = __shfl_sync(0xffffffffu, mine.bias, from);
                q.inv = __shfl_sync(0xffffffffu, mine.inv, from);
                word[g] = kv_quant_q4(next[i][g], q);
            }
            store(i, word, nullptr);
            __syncwarp();
        }
        // lane w has the parameters of pass w / 2, group w % 2 (or K's and V's)
        const int from = w / NW * WR + lane / X::LR, page = __shfl_sync(0xffffffffu, to, from), p = __shfl_sync(0xffffffffu, at, from);
        if (page >= 0)
            *reinterpret_cast<uint32_t *>((w % NW == 0 ? ps[0] : ps[A - 1]) + kv_row(a.c, page, h, p) * (4 * NG) + (A == 2 ? 0 : w % NW * 4)) = mine.par;
    } else {
#pragma unroll 1  // once in the instruction cache
        for (int i = 0; i < a.passes; ++i) {
            uint4 u[NW];
#pragma unroll
            for (int g = 0; g < NW; ++g) u[g] = next[0][g];
            if (i + 1 < a.passes) fetch(t0 + (i + 1) * X::R, true, next[0]);
            uint32_t word[NW], par[NW];
#pragma unroll
            for (int g = 0; g < NW; ++g) word[g] = kv_quant_fp4(u[g], par[g]);
            store(i, word, par);
            __syncwarp();
        }
    }
}

template <int FMT, int D>
__global__ void __launch_bounds__(128) k_kv_read(const KvReadArgs a) {
    using X = Wd<FMT, D>;
    constexpr int NG = X::NG, A = X::A;
    using T = typename Vec<NG>::T;
    const int w = threadIdx.x % X::LR, h = A == 2 ? blockIdx.y : blockIdx.y >> 1;
    const bool isv = A == 1 && (blockIdx.y & 1);
    const int t0 = (int)blockIdx.x * (X::R * a.passes) + (int)threadIdx.x / X::LR;
    const uint32_t *codes[A];
    const unsigned char *ps[A];
    uint16_t *dst[A];
#pragma unroll
    for (int x = 0; x < A; ++x) {
        const bool v = isv || x == 1;
        codes[x] = (v ? a.c.vq : a.c.kq) + w * NG;
        ps[x] = static_cast<const unsigned char *>(v ? a.c.vs : a.c.ks);
        dst[x] = (v ? a.v : a.k) + (size_t)h * D + 8 * w;
    }
    pdl_wait();
    uint32_t code[KV_U][A][NG], par[KV_U][A][FMT == FMT_Q4 ? NG : 1];
    int has = 0, got = 0;  // bit i: row i is some sequence's, its page is valid
    int r0 = 0, r1 = 0, b = -1;
#pragma unroll
    for (int i = 0; i < KV_U; ++i) {
        const int t = t0 + i * X::R;
        if (t >= a.s.T || i >= a.passes) continue;
        if (t >= r1 || t < r0) b = kv_seq_of(a.s, t, r0, r1);
        if (b < 0) continue;
        has |= 1 << i;
        const long p = (long)(a.first ? a.first[b] : 0) + (t - r0);
        const long page = p >= 0 && p <= 0x7fffffffL ? kv_page(a.c, a.s, b, (int)p) : -1;
        if (page < 0) {
            if (w == 0) atomicOr(a.c.err, ERR_PAGE);
            continue;
        }
        got |= 1 << i;
        const size_t row = kv_row(a.c, page, h, (int)p);
#pragma unroll
        for (int x = 0; x < A; ++x) {
            *reinterpret_cast<T *>(code[i][x]) = *reinterpret_cast<const T *>(codes[x] + row * (D / 8));
            if (FMT == FMT_Q4) *reinterpret_cast<T *>(par[i][x]) = *reinterpret_cast<const T *>(ps[x] + row * (4 * NG));
            else par[i][x][0] = NG == 4 ? *reinterpret_cast<const uint32_t *>(ps[x] + row * NG) : *reinterpret_cast<const uint16_t *>(ps[x] + row * NG);
        }
    }
#pragma unroll
    for (int i = 0; i < KV_U; ++i) {
        if (!((has >> i) & 1)) continue;
#pragma unroll
        for (int x = 0; x < A; ++x) {
            uint32_t word[NG];
            lane_words<FMT>(code[i][x], word, true);
            uint16_t *to = dst[x] + (size_t)(t0 + i * X::R) * a.c.Hkv * D;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float y[8];
                kv_word_values<FMT>(word[g], FMT == FMT_Q4 ? par[i][x][FMT == FMT_Q4 ? g : 0] : (par[i][x][0] >> (8 * g)) & 255u, y);
                const uint4 o = make_uint4(pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]), pack_bf2(y[4], y[5]), pack_bf2(y[6], y[7]));
                *reinterpret_cast<uint4 *>(to + g * (8 * X::LR)) = (got >> i) & 1 ? o : make_uint4(0, 0, 0, 0);
            }
        }
    }
}

#define KV_INST(F, D)                                \
    template __global__ void k_kv_write<F, D>(const KvWriteArgs); \
    template __global__ void k_kv_read<F, D>(const KvReadArgs);
KV_INST(FMT_Q4, 64)
KV_INST(FMT_Q4, 128)
KV_INST(FMT_FP4, 64)
KV_INST(FMT_FP4, 128)

}  // namespace moeb
