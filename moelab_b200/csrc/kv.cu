// Writing K and V rows into the 4-bit cache, and reading them back (layout: kv.cuh). Both are one pass over memory:
// one thread per code word (8 values: a 16-byte load or store of bf16), the lanes of a group (8 for int4's 64 values, 4
// for MXFP4's 32) reduce its extremes by shuffles.
#include "kv.cuh"

namespace moeb {

// Quantizes 8 values of a group spread over LANES neighbouring lanes, operation for operation as the weight quantizers
// (quant.cu), so a cache row equals mx.quantize of it. A group that holds an infinity or a NaN, or whose span passes
// fp32, is stored with NaN parameters: it reads back as NaN everywhere, and nothing else is touched by it.
MOEB_DEV uint32_t kv_quant_q4(const float (&v)[8], uint32_t &par) {
    float hi = v[0], lo = v[0];
    bool bad = !(fabsf(v[0]) <= 3.4028234e38f);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        hi = fmaxf(hi, v[i]);
        lo = fminf(lo, v[i]);
        bad |= !(fabsf(v[i]) <= 3.4028234e38f);
    }
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    const unsigned group = 0xffu << (threadIdx.x & 24);
    bad = (__ballot_sync(0xffffffffu, bad) & group) != 0;
    const bool mask = fabsf(lo) > fabsf(hi);
    float scale = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
    bad |= !(scale <= 3.4028234e38f);
    scale = scale > 1e-7f ? scale : 1e-7f;
    scale = mask ? scale : -scale;
    const float edge = mask ? lo : hi;
    const float q0 = rintf(__fdiv_rn(edge, scale));
    float bias = 0.0f;
    if (q0 != 0.0f) {
        scale = __fdiv_rn(edge, q0);
        bias = edge;
    }
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float q = rintf(__fdiv_rn(__fsub_rn(v[i], bias), scale));
        q = fminf(fmaxf(q, 0.0f), 15.0f);
        word |= (uint32_t)q << (4 * ((i >> 1) + 4 * (i & 1)));
    }
    // q0 = 0: the largest magnitude is below half the smallest scale, every code is 0 and the values are zeros. The weight
    // quantizer keeps that scale; here it is 0, so that attention, which takes codes less 8, meets nothing to cancel.
    par = bad ? 0x7fff7fffu : q0 == 0.0f ? 0u : (uint32_t)f2bf(scale) | ((uint32_t)f2bf(bias) << 16);
    return bad ? 0u : word;
}
MOEB_DEV uint32_t kv_quant_fp4(const float (&v)[8], uint32_t &par) {
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
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(__fmul_rn(v[i], inv));
        uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
        c |= (__float_as_uint(v[i]) >> 28) & 8u;
        word |= c << (4 * i);
    }
    return word;
}

template <int FMT, int D>
__global__ void __launch_bounds__(128) k_kv_write(KvWriteArgs a) {
    constexpr int W = D / 8;
    pdl_wait();
    const long gid = (long)blockIdx.x * blockDim.x + threadIdx.x;
    const int w = (int)(gid % W);
    long r = gid / W;  // (t, K or V, h), h fastest
    const int h = (int)(r % a.c.Hkv);
    r /= a.c.Hkv;
    const bool isv = (r & 1) != 0;
    const long t = r >> 1;
    long page = -1;
    int p = -1;
    if (t < a.s.T) {
        int r0, r1;
        const int b = kv_seq_of(a.s, (int)t, r0, r1);
        if (b >= 0) p = a.s.lens[b] - (r1 - (int)t);
        if (p >= 0) {
            page = kv_page(a.c, a.s, b, p);
            if (page < 0 && w == 0) atomicOr(a.c.err, ERR_PAGE);
        }
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (page >= 0) {
        const uint16_t *src = isv ? a.v + t * a.v_row + h * a.v_head : a.k + t * a.k_row + h * a.k_head;
        const uint4 u = *reinterpret_cast<const uint4 *>(src + 8 * w);
        const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = bf16lo(uu[i]);
            x[2 * i + 1] = bf16hi(uu[i]);
        }
    }
    // every lane takes part in the shuffles; a group's lanes are all inside one row
    uint32_t par;
    const uint32_t word = FMT == FMT_Q4 ? kv_quant_q4(x, par) : kv_quant_fp4(x, par);
    if (page < 0) return;
    const size_t row = kv_row(a.c, page, h, p);
    uint32_t *codes = isv ? a.c.vq : a.c.kq;
    if (FMT == FMT_Q4) {
        codes[row * W + kv_pos_q4<D>(w)] = word;
    } else {
        uint16_t *dst = reinterpret_cast<uint16_t *>(codes) + row * (D / 4);
        dst[kv_pos_fp4<D>(2 * w)] = (uint16_t)word;
        dst[kv_pos_fp4<D>(2 * w + 1)] = (uint16_t)(word >> 16);
    }
    void *ps = isv ? a.c.vs : a.c.ks;
    if (FMT == FMT_Q4) {
        if ((w & 7) == 0) static_cast<uint32_t *>(ps)[row * (D / 64) + (w >> 3)] = par;
    } else if ((w & 3) == 0) {
        static_cast<uint8_t *>(ps)[row * (D / 32) + (w >> 2)] = (uint8_t)par;
    }
}

template <int FMT, int D>
__global__ void __launch_bounds__(128) k_kv_read(KvReadArgs a) {
    constexpr int W = D / 8;
    pdl_wait();
    const long gid = (long)blockIdx.x * blockDim.x + threadIdx.x;
    const int w = (int)(gid % W);
    long r = gid / W;
    const int h = (int)(r % a.c.Hkv);
    r /= a.c.Hkv;
    const bool isv = (r & 1) != 0;
    const long t = r >> 1;
    if (t >= a.s.T) return;
    int r0, r1;
    const int b = kv_seq_of(a.s, (int)t, r0, r1);
    if (b < 0) return;
    const long p = (long)(a.first ? a.first[b] : 0) + (t - r0);
    const long page = p >= 0 && p <= 0x7fffffffL ? kv_page(a.c, a.s, b, (int)p) : -1;
    uint4 o = make_uint4(0, 0, 0, 0);
    if (page >= 0) {
        const size_t row = kv_row(a.c, page, h, (int)p);
        const uint32_t word = kv_word<FMT, D>(isv ? a.c.vq : a.c.kq, row, w);
        float x[8];
        kv_word_values<FMT>(word, kv_par<FMT>(isv ? a.c.vs : a.c.ks, row, w, D), x);
        o = make_uint4(pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(x[4], x[5]), pack_bf2(x[6], x[7]));
    } else if (w == 0) {
        atomicOr(a.c.err, ERR_PAGE);
    }
    *reinterpret_cast<uint4 *>((isv ? a.v : a.k) + ((size_t)t * a.c.Hkv + h) * D + 8 * w) = o;
}

#define KV_INST(F, D)                                \
    template __global__ void k_kv_write<F, D>(KvWriteArgs); \
    template __global__ void k_kv_read<F, D>(KvReadArgs);
KV_INST(FMT_Q4, 64)
KV_INST(FMT_Q4, 128)
KV_INST(FMT_FP4, 64)
KV_INST(FMT_FP4, 128)

}  // namespace moeb
