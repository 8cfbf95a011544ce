// Attention of a few query rows per sequence over the 4-bit cache: decode steps and drafted tokens (layout: kv.cuh).
//
// y = sum_j w_j v_j / sum_j w_j, w_j = 2^(score_j - m), score = scale log2(e) q . k: one pass over the keys with a running
// maximum m (the sums so far are scaled when it grows), statistics and sums in fp32.
//
// The rows of a sequence that share a KV head (n tokens x Gq query heads, at most NC = 8 or 16) are the columns of
// one tensor-core tile, so the cache is read once for all of them. Long caches are bound by their bytes, short ones
// by the chain lengths -> page table -> codes -> sums. Measured:
//   64 sequences of 1 to 8192 tokens, 32 query heads on 8, int4 (306 MB): 86 us with the join, 3.6 TB/s; in its loop over the
//     blocks the kernel moves 5.9 TB/s (a copy 6.56), the rest is the 2 us until a CTA knows its run, the 5 us until its first
//     copies are there, CTAs that end between 59 and 78 us (memory is not equally far from all SMs) and the join. Shares of two
//     sizes, the small ones for CTAs that end early, cost more than they even out (92 against 85 us): new CTAs start slowly
//     under load. MXFP4: 88 us
//   one of 200,001 tokens, 64 heads on 4, MXFP4 (109 MB, two column tiles, 8 warps per SM): 53 us, 2.1 TB/s, bound by the
//     latencies of one warp's steps: half of the issue slots are taken
//   one of 1021 tokens, 32 heads on 4, int4: 7.4 us in a graph
//   16 of 8192 with 4 drafted rows each, 32 heads on 8 (two column tiles), int4: 70 us, 2.2 TB/s
//
// Work split: the visible keys of every (sequence, KV head) are cut into blocks of 128; all blocks of the call in a row are
// dealt to the CTAs in equal runs, so uneven lengths cost nothing and the host needs to know none of them (a captured
// graph replays with other lengths). A run's start and end cost about as much as FR blocks, which each (sequence, head) has
// in the count before its first one (without them CTAs with many short sequences end last: 106 us for the batch above). A CTA
// that holds all blocks of a (sequence, head) writes y; otherwise it leaves its unnormalised sum, maximum and sum of weights,
// and k_kv_attn_join joins them. Where the page tables' width or the window bounds the keys to a few blocks there is no second
// launch: a CTA (a.direct = 1) or a cluster of 8 CTAs, which join through their shared memories, has a (sequence, head)
// (1021 tokens: 8.4 us with the second launch; windows of 128: 26 us, 16 without).
//
// A warp takes 32 keys of each block, straight from a cp.async ring of its own (no block-wide barrier in the loop; the next
// run's first copies are on their way while a run's warps join; bulk copies from single lanes cost twice the instructions), and
// feeds the codes to mma.sync m16n8k16 without dequantizing them. mma.sync and not tcgen05: its pipe is busy for a fifth of
// the time, and codes would have to be written to shared or tensor memory once more on their way.
//   scores^T [16 keys x NC] = K codes . q, q in fp16 after a power of two per row (8 bits of significand fit 11). int4: a
//     masked code is an fp16 subnormal, code * 2^-24, so that an operand costs one instruction (converted: 114 us for the batch
//     above when that was 106); with group g's scale s and bias b, score = sum_g s acc_g + b qsum_g in fp32. MXFP4: E2M1 codes
//     convert to fp16, score = sum_g 2^e acc_g.
//   y^T [D x NC] += V^T codes . P, P = fp16(p * scale of the key's group). A running power of two per warp, taken into p's
//     exponent, keeps the product in fp16's range whatever the values' size; codes as subnormals (int4) or E2M1 in fp16 are
//     exact. fp16 and not bf16: P is the only rounding here, 2^-11 keeps it below the result's own 2^-8. int4's bias term is
//     summed in fp32.
// A column's maximum is shared by the warp's lanes (three shuffles), warps join at the end of a run of blocks. MMA row r is key
// r / 2 + 4 (r % 2) of its eight, which makes the four keys of a lane's V operand consecutive rows of shared memory (no bank
// conflicts) and costs K nothing.
#include <type_traits>

#include "kv.cuh"

namespace moeb {

namespace {

constexpr int FW = 4, FT = 32 * FW;  // warps per CTA, threads
constexpr int FS = 3;                // ring stages (4: two CTAs per SM instead of three, 96 us for the batch above)
constexpr int FB = 32 * FW;          // keys per block
constexpr int FR = 2;                // blocks that a run costs besides its own
constexpr float LEAST = 1.2e-38f;    // a column's scale at least

template <int FMT, int D>
struct Few {
    static constexpr int G = D / 64, NG = FMT == FMT_Q4 ? D / 64 : D / 32;
    static constexpr int ROW = D / 2, PROW = FMT == FMT_Q4 ? G * 4 : NG;  // bytes of a row's codes, of its parameters
    static constexpr int O_V = 32 * ROW, O_KP = 2 * O_V, O_VP = O_KP + 32 * PROW, STAGE = O_VP + 32 * PROW;  // 32 rows
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
MOEB_DEV float h2_sum(uint32_t v) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&v));
    return f.x + f.y;
}
MOEB_DEV uint32_t h2_mul(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
MOEB_DEV uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// A key's parameters in fp32. int4: scale and bias; MXFP4: the powers of two.
template <int FMT, int NG>
MOEB_DEV void few_params(const unsigned char *p, float (&s)[NG], float (&b)[NG]) {
    if (FMT == FMT_Q4) {
        uint32_t w[2];
        if (NG == 2) {
            const uint2 x = *reinterpret_cast<const uint2 *>(p);
            w[0] = x.x;
            w[1] = x.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            s[g] = bf16lo(w[g]);
            b[g] = bf16hi(w[g]);
        }
    } else {
        const uint32_t w = NG == 4 ? *reinterpret_cast<const uint32_t *>(p) : *reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int g = 0; g < NG; g += 2) {
            e8m0_2(w >> (8 * g), s[g], s[g + 1]);
            b[g] = b[g + 1] = 0.f;
        }
    }
}
MOEB_DEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// from CTA `rank` of the cluster, at this CTA's shared address
MOEB_DEV float4 cluster_ld4(unsigned addr, unsigned rank) {
    float4 v;
    asm volatile("{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %4, %5;\n ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r];\n}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr), "r"(rank)
                 : "memory");
    return v;
}
MOEB_DEV float2 cluster_ld2(unsigned addr, unsigned rank) {
    float2 v;
    asm volatile("{\n .reg .b32 r;\n mapa.shared::cluster.u32 r, %2, %3;\n ld.shared::cluster.v2.f32 {%0, %1}, [r];\n}"
                 : "=f"(v.x), "=f"(v.y)
                 : "r"(addr), "r"(rank)
                 : "memory");
    return v;
}
MOEB_DEV void few_copy(unsigned smem, const unsigned char *gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
// int4 codes of nibble P of both halves of t as f16x2 subnormals: code * 2^-24 (P even) or code * 2^-20 (P odd), exact and
// without an operation on them but the mask
template <int P>
MOEB_DEV uint32_t q4_sub(uint32_t t) {
    return (P & 2 ? t >> 8 : t) & (P & 1 ? 0x00F000F0u : 0x000F000Fu);
}

// One sequence as the kernels see it: its rows, and the blocks of FB keys that any of them sees.
struct FewSeq {
    int r0, n, L, lo, ns, nb;
};
// End of the keys that a sequence of L tokens can have: its page table's, where that is shorter. It is a multiple of 16 then, so
// that no half of 16 keys is cut by it, and the kernel need not look at it per key.
MOEB_DEV int few_end(const KvAttnArgs &a, int L) { return min(L, a.s.P << a.c.pshift); }
// blocks [0, ns): the first tokens; then from lo / FB on. A sequence with rows has at least one block (its rows are
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
    q.ns = min((min(a.sinks, q.lo) + FB - 1) / FB, q.lo / FB);
    q.nb = q.n > 0 && (long)q.n * a.Gq <= a.few ? max(q.ns + max((few_end(a, q.L) + FB - 1) / FB - q.lo / FB, 0), 1) : 0;
    return q;
}
MOEB_DEV int few_units(const FewSeq &q) { return q.nb ? q.nb + FR : 0; }  // of each of its heads
MOEB_DEV int few_tok(const FewSeq &q, int k) { return (k < q.ns ? k : q.lo / FB + k - q.ns) * FB; }
// first unit of CTA c when W units are dealt to n CTAs: floor(W c / n), with divisions of 32 bits for all but huge calls
MOEB_DEV long few_start(long W, unsigned c, unsigned n) {
    if (W >> 32) return W * c / n;
    const unsigned w = (unsigned)W, q = w / n, r = w - q * n;
    return (long)q * c + r * c / n;
}

}  // namespace

// CTAs per SM: as many as registers allow without spills in the loop. Heads of 64 with one column tile: four (126 registers) and
// not three make many short windows faster (512 tokens in windows of 128, 64 heads on 8: 50 -> 42 us, 44 since values' sizes are
// looked at) and cost long caches nothing.
// ws: prefix[B + 1] int32 (blocks before each sequence), then 2 partials per CTA: NC rows of D sums, NC (max, sum).
template <int FMT, int D, int NT>
__global__ void __launch_bounds__(FT, NT == 1 ? (D == 64 ? 4 : 3) : D == 64 ? 3 : 2) k_kv_attn_few(const KvAttnArgs a, int *pre, float *part) {
    using F = Few<FMT, D>;
    constexpr int NC = 8 * NT, NG = F::NG;
    // The queries' operands stay in shared memory where that leaves registers for a third CTA per SM (two tiles of columns of
    // 128 values need two CTAs' share all the same: in 168 registers they spill, 200001 tokens 77 against 52 us).
    constexpr bool QS = NT == 2 && D == 64;
    extern __shared__ __align__(128) unsigned char sm[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
    unsigned char *ring = sm + warp * (FS * F::STAGE);
    float *so = reinterpret_cast<float *>(sm + FW * FS * F::STAGE);  // [FW][NC][D]
    uint4 *sq = reinterpret_cast<uint4 *>(so + FW * NC * D);
    __shared__ float s_m[FW][NC], s_l[FW][NC];
    __shared__ int s_sum[FW], s_b, s_pre;
    pdl_wait();

    int b, h, k0, k1;
    FewSeq q;
    long us = 0, ue = 0, seg = 0;  // this CTA's units; the first unit of its run's (sequence, head)
    // blocks [k0, k1) of the next run; a CTA whose share of a (sequence, head) is in its FR has none of its blocks
    auto locate = [&](bool next) {
        for (;; next = true) {
            if (next) {
                seg += q.nb + FR;
                if (++h == a.c.Hkv) {
                    h = 0;
                    do q = few_seq<NC>(a, ++b);
                    while (q.nb == 0);
                }
            }
            k0 = (int)max(us - seg - FR, 0L);
            k1 = (int)min(ue - seg - FR, (long)q.nb);
            if (k1 > k0 || ue <= seg + q.nb + FR) return;
        }
    };
    const unsigned rank = a.direct ? blockIdx.x % a.direct : 0;
    if (a.direct) {
        const unsigned i = blockIdx.x / a.direct;
        b = i / a.c.Hkv;
        h = i - b * a.c.Hkv;
        q = few_seq<NC>(a, b);
        if (rank == 0 && h == 0 && threadIdx.x == 0 && a.only && (long)q.n * a.Gq > a.few) atomicOr(a.c.err, ERR_ROWS);
        if (rank == 0 && h == 0 && threadIdx.x == 0 && q.nb && few_end(a, q.L) < q.L) atomicOr(a.c.err, ERR_PAGE);
        if (q.nb == 0) return;  // the whole cluster
        k0 = (int)((unsigned)q.nb * rank / a.direct);
        k1 = (int)((unsigned)q.nb * (rank + 1) / a.direct);
    } else {
        // every sequence's blocks: prefix sums over the CTA's threads, and the sequence of this CTA's first block
        const int per = (a.s.B + FT - 1) / FT, bb0 = min((int)threadIdx.x * per, a.s.B), bb1 = min(bb0 + per, a.s.B);
        int mine = 0;
        for (int b = bb0; b < bb1; ++b) mine += few_units(few_seq<NC>(a, b));
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
        const long units = (long)total * a.c.Hkv;
        const unsigned nct = (unsigned)min((long)gridDim.x, units);
        if (blockIdx.x == 0) {
            int at = base;
            for (int b = bb0; b < bb1; ++b) {
                const FewSeq s = few_seq<NC>(a, b);
                pre[b] = at;
                at += few_units(s);
                if (s.nb && few_end(a, s.L) < s.L) atomicOr(a.c.err, ERR_PAGE);  // tokens that the table has no place for
                if (a.only && (long)s.n * a.Gq > a.few) atomicOr(a.c.err, ERR_ROWS);
            }
            if (threadIdx.x == 0) pre[a.s.B] = total;
        }
        if (blockIdx.x >= nct) return;
        us = few_start(units, blockIdx.x, nct);
        ue = few_start(units, blockIdx.x + 1, nct);
        const long u = us;
        if (u >= (long)base * a.c.Hkv && u < (long)(base + mine) * a.c.Hkv) {
            int at = base, x = bb0;
            for (;; ++x) {
                const int nb = few_units(few_seq<NC>(a, x));
                if (u < (long)(at + nb) * a.c.Hkv) break;
                at += nb;
            }
            s_b = x;
            s_pre = at;
        }
        __syncthreads();
        b = s_b;
        q = few_seq<NC>(a, b);
        seg = (long)s_pre * a.c.Hkv;
        h = us - seg < 0x7fffffffL ? (int)((unsigned)(us - seg) / (unsigned)(q.nb + FR)) : (int)((us - seg) / (q.nb + FR));
        seg += (long)h * (q.nb + FR);
        locate(false);
        if (k1 <= k0) return;
    }
    const int ta = (r >> 1) + 4 * (r & 1);  // this lane's keys of 16: ta and ta + 8

    // Page ids of 16 blocks from kb on: lane 2 i + x has half x (16 keys, a page at least) of this warp's keys of block kb + i.
    // -1: no row sees the half; -2: it has no page.
    auto pages = [&](const FewSeq &q, int b, int kb, int k1) {
        const int k = kb + (lane >> 1), tok = few_tok(q, k) + 32 * warp + 16 * (lane & 1);
        if (k >= k1 || tok >= few_end(a, q.L) || (tok + 15 < q.lo && tok >= a.sinks)) return -1;
        const long page = kv_page(a.c, a.s, b, tok);
        return page < 0 ? -2 : (int)page;
    };
    // Copies of this warp's 32 keys of block k of head h. ok: bit 2 s + x says that half x of stage s has come. Addresses are
    // the lane's place in the arrays' first page, and one 64-bit product for codes and one for parameters per half.
    unsigned ok = 0;
    int slot_in = 0, slot = 0;  // stage of the next copy, of the next use
    const unsigned per_page = (unsigned)a.c.Hkv << a.c.pshift, pmask = (1u << a.c.pshift) - 1u;  // rows
    const unsigned char *kq = reinterpret_cast<const unsigned char *>(a.c.kq) + lane * 16, *vq = reinterpret_cast<const unsigned char *>(a.c.vq) + lane * 16;
    // lanes 0 .. PROW - 1: K's parameters, the next as many V's
    const bool parv = lane >= F::PROW;
    const unsigned char *pq = static_cast<const unsigned char *>(parv ? a.c.vs : a.c.ks) + (parv ? lane - F::PROW : lane) * 16;
    const unsigned st0 = smem_u32(ring) + lane * 16, sp0 = smem_u32(ring) + (parv ? F::O_VP + (lane - F::PROW) * 16 : F::O_KP + lane * 16);
    auto issue = [&](const FewSeq &q, int h, int k, int k1, int ids, int kb) {
        if (k < k1) {
            const unsigned row0 = ((unsigned)h << a.c.pshift) + ((unsigned)(few_tok(q, k) + 32 * warp) & pmask);
            const unsigned stage = slot_in * F::STAGE;
            unsigned has = 0;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int page = __shfl_sync(0xffffffffu, ids, 2 * (k - kb) + x);
                if (page < 0) {
                    if (page == -2 && lane == 0) atomicOr(a.c.err, ERR_PAGE);
                    continue;
                }
                has |= 1u << x;
                // a page of 16 keys: the second half starts at its page's first row
                const unsigned row = x == 0 ? row0 : ((unsigned)h << a.c.pshift) + ((unsigned)(few_tok(q, k) + 32 * warp + 16) & pmask);
                const size_t at = (size_t)(unsigned)page * per_page + row;
                const unsigned char *ks = kq + at * F::ROW, *vs = vq + at * F::ROW;
                const unsigned st = st0 + stage + x * (16 * F::ROW);
#pragma unroll
                for (int i = 0; i < F::ROW / 32; ++i) {
                    few_copy(st + i * 512, ks + i * 512);
                    few_copy(st + F::O_V + i * 512, vs + i * 512);
                }
                if (lane < 2 * F::PROW) few_copy(sp0 + stage + x * (16 * F::PROW), pq + at * F::PROW);
            }
            ok = (ok & ~(3u << (2 * slot_in))) | has << (2 * slot_in);
            if (++slot_in == FS) slot_in = 0;
        }
        cp_commit();
    };
    int kb = k0;
    int ids = pages(q, b, kb, k1);
#pragma unroll 1
    for (int i = 0; i < FS; ++i) issue(q, h, k0 + i, k1, ids, kb);

    while (true) {
        // ---- one run of blocks [k0, k1) of (b, h), whose first copies are on their way
        const int p0 = q.L - q.n, plast = q.L - 1;  // positions of the first and the last row
        // the next run: where it is and its first page ids, in time for its copies
        const FewSeq qr = q;
        const int hr = h, kr0 = k0, kr1 = k1;
        const long segr = seg;
        const int br = b;
        bool more = !a.direct && ue > seg + q.nb + FR;
        int idn = -1;
        if (more) {
            locate(true);
            more = k1 > k0;
            if (more) idn = pages(q, b, k0, k1);
        }
        // ---- queries: column nt * 8 + r is row (column / Gq) of the sequence, head h * Gq + column % Gq
        uint32_t qf[NT][D / 16][2];
        float qs[NT][FMT == FMT_Q4 ? NG : 1][2], cs[NT][2];
        int pos[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int col = nt * 8 + r, i = kv_div(col, a.Gdiv);
            const bool have = i < qr.n;
            const uint16_t *src = a.q + (have ? (qr.r0 + i) * a.q_row + (hr * a.Gq + col - i * a.Gq) * a.q_head : 0);
            uint4 w[D / 32];
            // words of this lane: int4 2 c, 2 c + 1 of every group of 64; MXFP4 c of every group of 32
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const int word = FMT == FMT_Q4 ? 8 * (j >> 1) + 2 * c + (j & 1) : 4 * j + c;
                w[j] = have ? *reinterpret_cast<const uint4 *>(src + 8 * word) : make_uint4(0, 0, 0, 0);
            }
            float qsum[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) qsum[g] = 0.f;
            // the scale's sign goes into q, so that the maximum can be taken before scaling; a scale of zero makes q zero
            const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
            float mul = a.scale == 0.f ? 1.f : fabsf(a.scale);
#pragma unroll
            for (int j = 0; j < D / 32; ++j)
                w[j] = a.scale == 0.f ? make_uint4(0, 0, 0, 0) : make_uint4(w[j].x ^ flip, w[j].y ^ flip, w[j].z ^ flip, w[j].w ^ flip);
            {  // to fp16 by the row's power of two: its largest value near 2^14 (int4), 2^8 (MXFP4)
                constexpr int UP = FMT == FMT_Q4 ? 14 : 8;
                uint32_t t16 = 0;
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const uint32_t ww[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) t16 = max(t16, max(ww[e] & 0x7fffu, (ww[e] >> 16) & 0x7fffu));
                }
                t16 = max(t16, __shfl_xor_sync(0xffffffffu, t16, 1));
                t16 = max(t16, __shfl_xor_sync(0xffffffffu, t16, 2));
                const int e = min(max((int)(t16 >> 7), UP + 1), 254);  // biased exponent of the largest value
                // 2^(UP - (e - 127)); a row that is not finite becomes NaN, as infinities would not where all scores are -inf
                const float down = t16 < 0x7f80u ? __uint_as_float((uint32_t)(254 + UP - e) << 23) : __uint_as_float(0x7fffffffu);
                // what undoes it; int4: and 2^24 for the codes, taken out of qsum below
                mul *= __uint_as_float((uint32_t)(e - UP) << 23) * (FMT == FMT_Q4 ? 16777216.f : 1.f);
                if (t16 == 0) mul = 1.f;
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    uint32_t ww[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) ww[x] = pack_h2(bf16lo(ww[x]) * down, bf16hi(ww[x]) * down);
                    if (FMT == FMT_Q4) {
                        qsum[j / 2 < NG ? j / 2 : 0] += h2_sum(ww[0]) + h2_sum(ww[1]) + h2_sum(ww[2]) + h2_sum(ww[3]);
                        // the odd pairs meet codes * 2^-20: words 1 and 3 hold values 2, 3 and 6, 7 of eight
                        ww[1] = h2_mul(ww[1], 0x2C002C00u);
                        ww[3] = h2_mul(ww[3], 0x2C002C00u);
                    }
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
                    float t = qsum[g] * 5.9604644775390625e-8f;  // 2^-24
                    t += __shfl_xor_sync(0xffffffffu, t, 1);
                    t += __shfl_xor_sync(0xffffffffu, t, 2);
                    qs[nt][g][0] = __shfl_sync(0xffffffffu, t, 8 * c);
                    qs[nt][g][1] = __shfl_sync(0xffffffffu, t, 8 * c + 4);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                cs[nt][e] = fmaxf(__shfl_sync(0xffffffffu, mul, 8 * c + 4 * e), LEAST);  // above zero: a hidden -inf stays -inf
                const int ce = nt * 8 + 2 * c + e, ie = kv_div(ce, a.Gdiv);
                pos[nt][e] = ie < qr.n ? p0 + ie : -1;  // a column without a row sees nothing
            }
        }

        if (QS) {  // the same for all warps
            if (warp == 0) {
#pragma unroll
                for (int x = 0; x < D / 16; ++x) sq[x * 32 + lane] = make_uint4(qf[0][x][0], qf[0][x][1], qf[NT - 1][x][0], qf[NT - 1][x][1]);
            }
            __syncthreads();
        }
        auto query = [&](int x, uint32_t (&f)[NT][2]) {  // operands of product x
            if (QS) {
                const uint4 v = sq[x * 32 + lane];
                f[0][0] = v.x;
                f[0][1] = v.y;
                f[NT - 1][0] = v.z;
                f[NT - 1][1] = v.w;
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    f[nt][0] = qf[nt][x][0];
                    f[nt][1] = qf[nt][x][1];
                }
            }
        };
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
        uint32_t low = ~0u;  // the smallest group of values among this lane's keys, less what counts as zero (which wraps)
        uint32_t vlim = 0;  // bits of the largest value scale that the running power of two takes
        float vexp = 0.f;   // its exponent: weights are 2^(score - m + vexp), and o, l and bs are sums of them

#pragma unroll 1
        for (int k = kr0; k < kr1; ++k) {
            cp_wait<FS - 1>();
            __syncwarp();
            const unsigned has = (ok >> (2 * slot)) & 3u;
            const unsigned char *st = ring + slot * F::STAGE;
            const int tok = few_tok(qr, k) + 32 * warp;
            const bool all = has == 3u && tok + 31 <= p0 && (!a.window || tok > plast - a.window || tok + 31 < a.sinks);
            // full: every row sees all 32 keys
            auto step = [&](auto full_) {
                constexpr bool full32 = decltype(full_)::value;
                // ---- scores of keys 16 x + ta, 16 x + ta + 8 for columns 2 c, 2 c + 1
                float s[2][NT][4];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[x][nt][0] = s[x][nt][1] = s[x][nt][2] = s[x][nt][3] = 0.f;
                    uint32_t wa[D / 32], wb[D / 32];
                    const unsigned char *ra = st + (16 * x + ta) * F::ROW + c * (D / 8);
                    if (D == 128) {
                        const uint4 y = *reinterpret_cast<const uint4 *>(ra), z = *reinterpret_cast<const uint4 *>(ra + 8 * F::ROW);
                        wa[0] = y.x; wa[1] = y.y; wa[D / 32 - 2] = y.z; wa[D / 32 - 1] = y.w;
                        wb[0] = z.x; wb[1] = z.y; wb[D / 32 - 2] = z.z; wb[D / 32 - 1] = z.w;
                    } else {
                        const uint2 y = *reinterpret_cast<const uint2 *>(ra), z = *reinterpret_cast<const uint2 *>(ra + 8 * F::ROW);
                        wa[0] = y.x; wa[1] = y.y;
                        wb[0] = z.x; wb[1] = z.y;
                    }
                    float xa[NG], ya[NG], xb[NG], yb[NG];
                    few_params<FMT, NG>(st + F::O_KP + (16 * x + ta) * F::PROW, xa, ya);
                    few_params<FMT, NG>(st + F::O_KP + (16 * x + ta + 8) * F::PROW, xb, yb);
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        float acc[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
                        if (FMT == FMT_Q4) {
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                const uint32_t ua = wa[(y >> 1) * NG + g], ub = wb[(y >> 1) * NG + g];
                                uint32_t A[4];
                                if (y & 1) { A[0] = q4_sub<2>(ua); A[1] = q4_sub<2>(ub); A[2] = q4_sub<3>(ua); A[3] = q4_sub<3>(ub); }
                                else { A[0] = q4_sub<0>(ua); A[1] = q4_sub<0>(ub); A[2] = q4_sub<1>(ua); A[3] = q4_sub<1>(ub); }
                                uint32_t f[NT][2];
                                query(4 * g + y, f);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) mma_f16(acc[nt], A, f[nt][0], f[nt][1]);
                            }
                        } else {
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
                            uint32_t f0[NT][2], f1[NT][2];
                            query(2 * g, f0);
                            query(2 * g + 1, f1);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma_f16(acc[nt], A0, f0[nt][0], f0[nt][1]);
                                mma_f16(acc[nt], A1, f1[nt][0], f1[nt][1]);
                            }
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                if (FMT == FMT_Q4) {
                                    s[x][nt][e] = fmaf(ya[g], qs[nt][FMT == FMT_Q4 ? g : 0][e], s[x][nt][e]);
                                    s[x][nt][2 + e] = fmaf(yb[g], qs[nt][FMT == FMT_Q4 ? g : 0][e], s[x][nt][2 + e]);
                                }
                                s[x][nt][e] = fmaf(xa[g], acc[nt][e], s[x][nt][e]);
                                s[x][nt][2 + e] = fmaf(xb[g], acc[nt][2 + e], s[x][nt][2 + e]);
                            }
                        }
                    }
                }
                {  // The smallest group of values, by its largest magnitude (int4: |bias|, 7.5 scales or more; the bits doubled to drop
                   // its sign) or its power of two. The four lanes that have the same keys below take one of the four keys each (all
                   // four in every lane: 88 us for the batch above; nothing looked at: 85)
                    const int j = 16 * (c >> 1) + 8 * (c & 1) + ta;
                    const unsigned char *par = st + F::O_VP + j * F::PROW;
                    if (full32 || (((has >> (c >> 1)) & 1u) && tok + j <= plast && (tok + j >= qr.lo || tok + j < a.sinks))) {
                        if (FMT == FMT_Q4) {
#pragma unroll
                            for (int g = 0; g < NG; ++g) low = min(low, 2u * reinterpret_cast<const uint32_t *>(par)[g] - 2u * KV_ZERO);
                        } else {
                            const uint32_t w = NG == 4 ? *reinterpret_cast<const uint32_t *>(par) : *reinterpret_cast<const uint16_t *>(par);
#pragma unroll
                            for (int g = 0; g < NG; ++g) low = min(low, __byte_perm(w, 0, 0x4440 + g) - (KV_ZERO >> 23));
                        }
                    }
                }
                // ---- the value parameters of the same keys (zero where no row sees the key: what lies there is not looked at)
                float va[2][NG], vb[2][NG], ba[2][NG], bb[2][NG];
                unsigned vis[NT];  // bit 4 x + 2 i + e: column 2 c + e sees key 16 x + ta + 8 i
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    few_params<FMT, NG>(st + F::O_VP + (16 * x + ta) * F::PROW, va[x], ba[x]);
                    few_params<FMT, NG>(st + F::O_VP + (16 * x + ta + 8) * F::PROW, vb[x], bb[x]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) vis[nt] = 0xffu;
                if (!full32) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int ja = tok + 16 * x + ta, jb = ja + 8;
                        const bool half = (has >> x) & 1u;
                        const bool sa = half && ja <= plast && (ja >= qr.lo || ja < a.sinks), sb = half && jb <= plast && (jb >= qr.lo || jb < a.sinks);
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            va[x][g] = sa ? va[x][g] : 0.f;
                            vb[x][g] = sb ? vb[x][g] : 0.f;
                            ba[x][g] = sa ? ba[x][g] : 0.f;
                            bb[x][g] = sb ? bb[x][g] : 0.f;
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int p = pos[nt][e];
                                const bool wa_ = half && ja <= p && (!a.window || ja > p - a.window || ja < a.sinks);
                                const bool wb_ = half && jb <= p && (!a.window || jb > p - a.window || jb < a.sinks);
                                if (!wa_) { s[x][nt][e] = -INFINITY; vis[nt] &= ~(1u << (4 * x + e)); }
                                if (!wb_) { s[x][nt][2 + e] = -INFINITY; vis[nt] &= ~(1u << (4 * x + 2 + e)); }
                            }
                        }
                    }
                }
                float big = 0.f;  // the largest scale; fmaxf passes NaN over
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int g = 0; g < NG; ++g) big = fmaxf(big, fmaxf(fabsf(va[x][g]), fabsf(vb[x][g])));
                const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
                float fix = 1.f;
                if (top > vlim) {  // larger than the power of two takes: scale to 2^8, with room to 2^14
                    const uint32_t e = min(max(top >> 23, 35u), 248u);
                    const float ne = (float)(135 - (int)e);
                    fix = ex2(ne - vexp);
                    vexp = ne;
                    vlim = (e + 6u) << 23;
                }
                // ---- running maximum, weights
                bool grew = fix != 1.f;
                float mn[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float t = fmaxf(fmaxf(s[0][nt][e], s[0][nt][2 + e]), fmaxf(s[1][nt][e], s[1][nt][2 + e]));
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                        mn[nt][e] = fmaxf(m[nt][e], t * cs[nt][e]);
                        grew |= mn[nt][e] > m[nt][e];
                    }
                }
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float f = ex2(m[nt][e] - (mn[nt][e] == -INFINITY ? 0.f : mn[nt][e])) * fix;
                            m[nt][e] = mn[nt][e];
                            l[nt][e] *= f;
                            if (FMT == FMT_Q4) {
#pragma unroll
                                for (int g = 0; g < NG; ++g) bs[nt][FMT == FMT_Q4 ? g : 0][e] *= f;
                            }
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) {
                                o[nt][i][e] *= f;
                                o[nt][i][2 + e] *= f;
                            }
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    uint32_t pf[NT][NG][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float off = m[nt][e] == -INFINITY ? 0.f : vexp - m[nt][e];
                            s[x][nt][e] = ex2(fmaf(s[x][nt][e], cs[nt][e], off));
                            s[x][nt][2 + e] = ex2(fmaf(s[x][nt][2 + e], cs[nt][e], off));
                            l[nt][e] += s[x][nt][e] + s[x][nt][2 + e];
                        }
                        const float(&w)[4] = s[x][nt];
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            const float xa = va[x][g], xb = vb[x][g];
                            float y[4] = {w[0] * xa, w[1] * xa, w[2] * xb, w[3] * xb};
                            if (!full32) {  // a key that one row sees and another does not may hold a NaN
#pragma unroll
                                for (int e = 0; e < 4; ++e) y[e] = (vis[nt] >> (4 * x + e)) & 1u ? y[e] : 0.f;
                            }
                            pf[nt][g][0] = transpose8(pack_h2(y[0], y[1]));
                            pf[nt][g][1] = transpose8(pack_h2(y[2], y[3]));
                            if (FMT == FMT_Q4) {
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    float &t = bs[nt][FMT == FMT_Q4 ? g : 0][e];
                                    if (full32) {
                                        t = fmaf(w[2 + e], bb[x][g], fmaf(w[e], ba[x][g], t));
                                    } else {
                                        t += (vis[nt] >> (4 * x + e)) & 1u ? w[e] * ba[x][g] : 0.f;
                                        t += (vis[nt] >> (4 * x + 2 + e)) & 1u ? w[2 + e] * bb[x][g] : 0.f;
                                    }
                                }
                            }
                        }
                    }
                    // ---- values: keys 16 x + c, + 4, + 8, + 12
                    const unsigned char *rv = st + F::O_V + (16 * x + c) * F::ROW + r * (D / 16);
                    uint32_t vw[4][D / 64];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        if (D == 128) {
                            const uint2 y = *reinterpret_cast<const uint2 *>(rv + t * 4 * F::ROW);
                            vw[t][0] = y.x;
                            vw[t][D / 64 - 1] = y.y;
                        } else {
                            vw[t][0] = *reinterpret_cast<const uint32_t *>(rv + t * 4 * F::ROW);
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
                                if (p == 0) { A[0] = q4_sub<0>(l0); A[1] = q4_sub<0>(h0); A[2] = q4_sub<0>(l1); A[3] = q4_sub<0>(h1); }
                                if (p == 1) { A[0] = q4_sub<1>(l0); A[1] = q4_sub<1>(h0); A[2] = q4_sub<1>(l1); A[3] = q4_sub<1>(h1); }
                                if (p == 2) { A[0] = q4_sub<2>(l0); A[1] = q4_sub<2>(h0); A[2] = q4_sub<2>(l1); A[3] = q4_sub<2>(h1); }
                                if (p == 3) { A[0] = q4_sub<3>(l0); A[1] = q4_sub<3>(h0); A[2] = q4_sub<3>(l1); A[3] = q4_sub<3>(h1); }
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
            };
            if (all) step(std::true_type{});
            else if (has) step(std::false_type{});
            __syncwarp();
            if (k + FS == kb + 16) {
                kb = k + FS;
                ids = pages(qr, br, kb, kr1);
            }
            issue(qr, hr, k + FS, kr1, ids, kb);
            if (++slot == FS) slot = 0;
        }
        // ---- the next run's first copies go out before this one's warps join
        if (more) {
#pragma unroll 1
            for (int i = 0; i < FS; ++i) issue(q, h, k0 + i, k1, idn, k0);
        }

        // ---- the warps' sums join in shared memory; m becomes what the weights are relative to
        bool far = false;  // scores so large that the product's rounding in m is one of whole powers of two in the weights
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                // or a query whose power of two and scale pass fp32
                far |= (fabsf(m[nt][e]) > KV_FAR && m[nt][e] != -INFINITY) || cs[nt][e] == LEAST || cs[nt][e] > 1e38f;
                m[nt][e] -= vexp;
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
        // a group of values too far below the largest for fp16? int4: |bias| is compared with the largest scale, an eighth of its own
        const int under = (int)(vlim >> 23) - (KV_SPREAD + 6 - (FMT == FMT_Q4 ? 3 : 0)) - (int)(KV_ZERO >> 23);
        const bool uneven = __syncthreads_or(far || (under > 0 && low < (FMT == FMT_Q4 ? (uint32_t)under << 24 : (uint32_t)under)));
        const bool whole = kr0 == 0 && kr1 == qr.nb;
        float *pt = part + ((size_t)blockIdx.x * 2 + (us >= segr ? 0 : 1)) * (NC * (D + 2));
        auto put = [&](int col, int d4, float4 v, float M, float L) {  // the run's sums of 4 values of a column
            if (a.direct > 1) {  // to the front of the rings, which are empty now
                float *mine = reinterpret_cast<float *>(sm);
                *reinterpret_cast<float4 *>(mine + col * D + 4 * d4) = v;
                if (d4 == 0) *reinterpret_cast<float2 *>(mine + NC * D + 2 * col) = make_float2(M, L);
            } else if (whole) {
                const int ri = kv_div(col, a.Gdiv), head = hr * a.Gq + col - ri * a.Gq;
                kv_finish<D>(a, qr.r0 + ri, head, d4, v, M, L);
            } else {
                *reinterpret_cast<float4 *>(pt + col * D + 4 * d4) = v;
                if (d4 == 0) *reinterpret_cast<float2 *>(pt + NC * D + 2 * col) = make_float2(M, L);
            }
        };
        if (uneven) {  // a warp per column, in fp32 from the cache
#pragma unroll 1
            for (int col = warp; col < qr.n * a.Gq; col += FW) {
                const int ri = kv_div(col, a.Gdiv);
                const KvSum x = kv_exact<FMT, D>(a, br, hr, a.q + (qr.r0 + ri) * a.q_row + (hr * a.Gq + col - ri * a.Gq) * a.q_head, p0 + ri, kr0,
                                                 kr1, qr.ns, qr.lo / FB - qr.ns);
                if (lane < D / 4) put(col, kv_dim<FMT, D>(lane) / 4, x.v, x.M, x.L);
            }
        } else {
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
                        const float up = FMT == FMT_FP4 ? 1.f : i & 1 ? 1048576.f : 16777216.f;  // codes were * 2^-20, 2^-24
                        v.x = fmaf(o[nt][i][e], up, add) * fm;
                        v.y = fmaf(o[nt][i][2 + e], up, add) * fm;
                        *reinterpret_cast<float2 *>(dst + dim) = v;
                    }
                }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < qr.n * a.Gq * (D / 4); i += FT) {
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
                put(col, d4, v, M, L);
            }
        }
        if (a.direct > 1) {
            // column i is CTA i % direct's: it adds up what all of them have
            cluster_sync();
            const unsigned at = smem_u32(sm);
            const int nc = qr.n * a.Gq, mine = ((int)(nc - rank) + a.direct - 1) / a.direct;  // columns of this CTA
            for (int i = threadIdx.x; i < mine * (D / 4); i += FT) {
                const int col = (int)rank + i / (D / 4) * a.direct, d4 = i % (D / 4);
                float M = -INFINITY, L = 0.f;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int x = 0; x < a.direct; ++x) M = fmaxf(M, cluster_ld2(at + (NC * D + 2 * col) * 4, x).x);
                const float use = M == -INFINITY ? 0.f : M;
                for (int x = 0; x < a.direct; ++x) {
                    const float2 ml = cluster_ld2(at + (NC * D + 2 * col) * 4, x);
                    const float4 w = cluster_ld4(at + (col * D + 4 * d4) * 4, x);
                    const float f = ex2(ml.x - use);
                    v.x += w.x * f;
                    v.y += w.y * f;
                    v.z += w.z * f;
                    v.w += w.w * f;
                    L += ml.y * f;
                }
                const int ri = kv_div(col, a.Gdiv);
                kv_finish<D>(a, qr.r0 + ri, hr * a.Gq + col - ri * a.Gq, d4, v, M, L);
            }
            cluster_sync();  // nobody leaves while its sums are read
        }
        if (!more) break;
        kb = k0;
        ids = idn;
        __syncthreads();
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
    const int at = pre[b], nu = pre[b + 1] - at, nb = nu - FR;
    if (nb < 2) return;  // none, or one block: one CTA had it
    const FewSeq q = few_seq<NC>(a, b);
    if (col >= q.n * a.Gq) return;
    const long units = (long)pre[a.s.B] * a.c.Hkv;
    const unsigned n = (unsigned)min((long)grid, units);
    const long seg = (long)at * a.c.Hkv + (long)h * nu, u0 = seg + FR, u1 = seg + nu;
    const int c0 = (int)(((u0 + 1) * n - 1) / units), c1 = (int)((u1 * n - 1) / units);  // CTAs of the first and last block
    if (c0 == c1) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int E = D / 32, SIZE = NC * (D + 2);
    // CTA x's partial: its first place when its share starts in this (sequence, head)
    auto partial = [&](int x) { return part + ((size_t)x * 2 + (few_start(units, x, n) >= seg ? 0 : 1)) * SIZE; };
    // the column's maximum first, so that the sums below do not wait for one another
    float M = -INFINITY;
    for (int x = c0 + (int)threadIdx.x; x <= c1; x += 256) M = fmaxf(M, partial(x)[NC * D + 2 * col]);
#pragma unroll
    for (int i = 16; i; i >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, i));
    if (lane == 0) s_m[warp] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) M = fmaxf(M, s_m[i]);
    const float use = M == -INFINITY ? 0.f : M;
    float l = 0.f, o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
#pragma unroll 4
    for (int x = c0 + warp; x <= c1; x += 8) {
        const float *pt = partial(x);
        const float2 ml = *reinterpret_cast<const float2 *>(pt + NC * D + 2 * col);
        const float f = ex2(ml.x - use);
        l += ml.y * f;
        const float *src = pt + col * D + lane * E;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] += src[i] * f;
    }
    if (lane == 0) s_l[warp] = l;
#pragma unroll
    for (int i = 0; i < E; ++i) so[warp][lane * E + i] = o[i];
    __syncthreads();
    if (threadIdx.x >= D / 4) return;
    float L = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 w = *reinterpret_cast<const float4 *>(&so[i][4 * threadIdx.x]);
        v.x += w.x;
        v.y += w.y;
        v.z += w.z;
        v.w += w.w;
        L += s_l[i];
    }
    const int ri = kv_div(col, a.Gdiv);
    kv_finish<D>(a, q.r0 + ri, h * a.Gq + col - ri * a.Gq, threadIdx.x, v, M, L);
}

template <int FMT, int D, int NT>
size_t kv_few_smem() {
    return (size_t)FW * FS * Few<FMT, D>::STAGE + (size_t)FW * 8 * NT * D * 4 + (NT == 2 && D == 64 ? D / 16 * 512 : 0);
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
