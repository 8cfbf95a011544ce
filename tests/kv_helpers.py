"""Shared by the 4-bit KV cache tests: batches of sequences with their pages, and the operators in 64 bits.

The reference takes the stored values from the oracle's quantizers (natural order, CPU) and computes attention from its
definition in float64; nothing of the library is on that path."""
import math

import numpy as np
import torch

import oracle

U_BF16, U_FP16 = 2.0 ** -8, 2.0 ** -11  # largest relative error of one rounding


def stored(w, fmt):
    """fp32 values that bf16 rows w [..., D] have in the cache (oracle quantizers)."""
    if fmt == "q4":
        return torch.from_numpy(oracle.q4_dequant(*oracle.q4_quantize(w)))
    return torch.from_numpy(oracle.mxfp4_dequant(*oracle.mxfp4_quantize(w)))


class Batch:
    """B sequences of the given lengths, the last rows[b] tokens of each being this call's. K / V of every token, a page
    table over shuffled pages (spare pages in between, -1 behind a sequence's end)."""

    def __init__(self, lens, rows, H, Hkv, D, fmt, page=16, seed=0, pad=0, device="cuda", peak=1.0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.rows, self.H, self.Hkv, self.D, self.fmt, self.page, self.pad = lens, rows, H, Hkv, D, fmt, page, pad
        self.device = device
        B, L = len(lens), max([1] + list(lens))
        gain = 0.5 + 1.5 * torch.rand(Hkv, D, generator=g)
        self.k = (torch.randn(B, L, Hkv, D, generator=g) * gain + 0.5 * torch.randn(Hkv, D, generator=g)).to(torch.bfloat16)
        self.v = (torch.randn(B, L, Hkv, D, generator=g) * (0.25 + torch.rand(B, L, Hkv, 1, generator=g))).to(torch.bfloat16)
        need = [-(-max(0, n) // page) for n in lens]
        self.pages = max(1, sum(need)) + spare
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((B, max([1] + need)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.table = self.table.to(device)
        self.lens_t = torch.tensor(lens, dtype=torch.int32, device=device)
        self.cu = torch.tensor([0] + list(np.cumsum(rows)), dtype=torch.int32, device=device)
        self.T = sum(rows) + pad
        self.q = (torch.randn(self.T, H, D, generator=g) * peak).to(torch.bfloat16).to(device)

    def cache(self, ops, fill=True):
        c = ops.KVCache(self.pages, self.Hkv, self.D, page_size=self.page, fmt=self.fmt, device=self.device)
        if fill:
            cu = torch.tensor([0] + list(np.cumsum(self.lens)), dtype=torch.int32, device=self.device)
            ops.kv_write(c, self.flat(self.k), self.flat(self.v), self.table, self.lens_t, cu=cu)
        return c

    def flat(self, x):
        """[tokens of all sequences, Hkv, D] of a [B, L, Hkv, D] tensor."""
        rows = [x[b, :n] for b, n in enumerate(self.lens)]
        return torch.cat(rows).contiguous().to(self.device)

    def new(self, x):
        """This call's rows of it (with the padding rows behind them)."""
        rows = [x[b, n - r:n] for b, (n, r) in enumerate(zip(self.lens, self.rows))]
        return torch.cat(rows + [torch.ones(self.pad, self.Hkv, self.D, dtype=x.dtype)]).contiguous().to(self.device)

    def reference(self, scale=None, window=0, sinks=0, sink_logits=None, hole=None):
        """(y, bound, lse) in float64: the definition, and how far the library's bf16 result may be from it.

        The bound. With A = sum_j p_j |v_j| / sum_j p_j: the result is rounded to bf16 (2^-8 of it). Inside, keys and values
        may be rounded to fp16 (2^-11 each, values relative to A; a key's moves a score by 2^-11 scale |q|.|k|), the
        probabilities to fp16 (2^-11, relative to A); fp32 sums and exp2 are below 2^-15 of A together with the score's own
        fp32 error, which with int4 codes offset by 128 is below 2^-20 * 136 * scale * s_max * |q|_1 (s_max: the largest
        step of int4, at most 2/15 of the largest |k|, so below 2^-11 scale |q|_1 max|k| / 7). A score moved by e moves the
        weighted mean by at most 2 e A.

        The probabilities' rounding, for int4: a value is s code + b, the second part is summed in fp32, so what a rounded p
        scales is s code, not the value: at most 15 s, and s <= (max - min) / 15 <= 2 / 15 of the group's largest |v|. So that
        term is 2^-11 sum_j p_j 2 max_group |v_j|, which is more than 2^-11 A where a value lies near zero in a group that does
        not (the step s of the stored value itself is 2^7 times that)."""
        scale = self.D ** -0.5 if scale is None else scale
        G = self.H // self.Hkv
        y = torch.zeros(self.T, self.H, self.D, dtype=torch.float64)
        bound = torch.zeros_like(y)
        lse = torch.full((self.T, self.H), -math.inf, dtype=torch.float64)
        ks, vs = stored(self.k, self.fmt).double().to(self.device), stored(self.v, self.fmt).double().to(self.device)
        q = self.q.double()
        at = 0
        for b, (L, n) in enumerate(zip(self.lens, self.rows)):
            pos = torch.arange(L - n, L, device=self.device)
            key = torch.arange(max(L, 0), device=self.device)
            see = key[None] <= pos[:, None]
            if window:
                see &= (key[None] > pos[:, None] - window) | (key[None] < sinks)
            if hole is not None and hole[0] == b:  # keys without a page
                see &= ~((key >= hole[1]) & (key < hole[2]))[None]
            for h in range(self.H):
                kk, vv, qq = ks[b, :L, h // G], vs[b, :L, h // G], q[at:at + n, h]
                s = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
                if sink_logits is not None:
                    s = torch.cat([s, sink_logits[h].double().to(self.device).expand(n, 1)], -1)
                if s.shape[1] == 0:
                    continue
                m = s.amax(-1, keepdim=True)
                p = torch.where(m == -math.inf, torch.zeros_like(s), torch.exp(s - torch.where(m == -math.inf, 0.0, m)))
                tot = p.sum(-1, keepdim=True)
                p = (p / torch.where(tot > 0, tot, 1.0))[:, :L]
                out = torch.where(p[:, :, None] > 0, p[:, :, None] * vv[None], 0.0).sum(1) if vv.isnan().any() else p @ vv
                y[at:at + n, h] = out.cpu()
                A = p @ vv.abs().nan_to_num()
                Ap = A
                if self.fmt == "q4":
                    top = vv.abs().nan_to_num().unflatten(-1, (-1, 64)).amax(-1, keepdim=True)
                    Ap = p @ top.expand(-1, -1, 64).flatten(1) * 2
                e = (qq.abs() @ kk.abs().T * scale).masked_fill(~see, 0.0).amax(-1, keepdim=True) if L else 0.0
                e = U_FP16 * e + U_FP16 / 7 * scale * qq.abs().sum(-1, keepdim=True) * (kk.abs().max() if L else 0.0)
                bound[at:at + n, h] = (U_BF16 * out.abs() + ((2 * e + U_FP16 + 2.0 ** -15) * A + U_FP16 * Ap) * (1 + U_BF16)).cpu() + 1e-30
                lse[at:at + n, h] = (m + torch.log(tot)).squeeze(-1).cpu()
            at += n
        return y, bound, lse


def check(y, ref, bound, what=""):
    y = y.double().cpu()
    assert torch.isfinite(y).all(), what
    off = (y - ref).abs() - bound
    assert (off <= 0).all(), (what, int((off > 0).sum()), off.max().item(), (off > 0).nonzero()[:4].tolist())
    if ref.numel() >= 1024 and ref.norm() > 0:
        # the roundings are independent: one to bf16 (2^-8 / sqrt(6) in the mean) and three to fp16 (2^-11 / sqrt(6) each,
        # the keys' at scores whose spread stays within the batch's), with half as much again for the spread of the mean
        rel = ((y - ref).norm() / ref.norm()).item()
        assert rel <= 1.5 * math.sqrt((U_BF16 ** 2 + 3 * (2 * U_FP16) ** 2) / 6), (what, rel)
