"""FP8 pools with a scale for each token and head, and attention over them in
64 bits with the room that a kernel's roundings take."""
from __future__ import annotations

import math

import torch

import fp8_ref

OUT_HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
W_HALF = 2.0 ** -11              # the weights of p.v are f16
NAN_CODE = 0x7F


class Pools:
    """Pools of N blocks whose unused slots hold NaN codes and NaN or infinite scales; sequence s has lens[s] tokens in
    shuffled blocks.  size: how much a row's magnitude varies (standard deviation of its natural logarithm)."""

    def __init__(self, lens, n_kv, BS, seed=0, size=0.5, v_factor=1.0, extra_blocks=2, max_blocks=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.n_kv, self.BS = list(lens), n_kv, BS
        counts = [(n + BS - 1) // BS for n in lens]
        self.N = sum(counts) + extra_blocks
        order = torch.randperm(self.N, generator=g, device="cuda").to(torch.int32)
        wide = max_blocks or max(1, max(counts, default=1))
        self.tables = torch.full((len(lens), wide), -1, dtype=torch.int32, device="cuda")
        shape = (self.N, n_kv, 128, BS)
        self.k, self.v = (torch.full(shape, NAN_CODE, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.ks = torch.full((self.N, n_kv, BS), float("nan"), device="cuda")
        self.vs = torch.full((self.N, n_kv, BS), float("inf"), device="cuda")
        at = 0
        for s, n in enumerate(counts):
            self.tables[s, :n] = order[at:at + n]
            for b in range(n):
                blk, m = int(order[at + b]), min(BS, lens[s] - b * BS)
                for codes, scales, f in ((self.k, self.ks, 1.0), (self.v, self.vs, v_factor)):
                    x = torch.randn(n_kv, 128, m, generator=g, device="cuda", dtype=torch.float64)
                    x *= torch.exp(size * torch.randn(n_kv, 1, m, generator=g, device="cuda", dtype=torch.float64)) * f
                    sc = (x.abs().amax(1) / fp8_ref.MAX).float()
                    codes[blk, :, :, :m] = (x / sc.double()[:, None]).clamp(-448, 448).float().to(
                        torch.float8_e4m3fn).view(torch.uint8)
                    scales[blk, :, :m] = sc
            at += n
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def rows(self, s, n):
        """k, v [n_kv, n, 128] of sequence s in float64, and which of its tokens lie in blocks that exist."""
        t = torch.arange(n, device="cuda")
        lb = t // self.BS
        there = lb < self.tables.shape[1]
        blk = self.tables[s, lb.clamp(max=self.tables.shape[1] - 1)].long()
        there = there & (blk >= 0) & (blk < self.N)
        blk, off = blk.clamp(0, self.N - 1), t % self.BS
        got = []
        for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
            x = fp8_ref.values(codes[blk, :, :, off]) * scales[blk, :, off].double()[..., None]    # [n, n_kv, 128]
            got.append(torch.where(there[:, None, None], x, torch.zeros_like(x)).transpose(0, 1).contiguous())
        return got[0], got[1], there

    def attention(self, q, s, n, scale, modulo=False):
        """q [rows, H, 128] at the last positions of sequence s's n tokens, causal: (out, room) [rows, H, 128]."""
        R, H, D = q.shape
        group = H // self.n_kv
        out, room = (torch.zeros(R, H, D, dtype=torch.float64, device="cuda") for _ in range(2))
        half = OUT_HALF[q.dtype]
        if n == 0:
            return out, room
        k, v, there = self.rows(s, n)
        seen = there[None, :] & (torch.arange(n, device="cuda")[None, :]
                                 <= (n - R + torch.arange(R, device="cuda"))[:, None])
        top_v = v.abs().amax(dim=(1, 2))
        for h in range(H):
            kv = h % self.n_kv if modulo else h // group
            x = q[:, h].double()
            sc = (x @ k[kv].t().contiguous() * scale).masked_fill(~seen, -math.inf)
            top = sc.amax(1, keepdim=True)
            live = torch.isfinite(top)
            w = torch.where(live, torch.exp(sc - torch.where(live, top, torch.zeros_like(top))), torch.zeros_like(sc))
            total = w.sum(1, keepdim=True).clamp(min=1e-300)
            p = w / total
            out[:, h] = p @ v[kv]
            spread = p @ v[kv].abs()
            # a score: 128 exact products added in fp32, the scales' products, the exponent's argument; twice, as
            # weights and their sum are both off by it
            off = (x.abs() @ k[kv].abs().t().contiguous() * scale).masked_fill(~seen, 0).amax(1, keepdim=True)
            off = 2 * (140 * fp8_ref.U32 * off + 2.0 ** -20)
            # weights rounded to f16, those of small scales to its subnormals; values rounded to f16 where a kernel
            # stages them; sums in fp32
            sub = n * 2.0 ** -24 * top_v[kv] / total
            room[:, h] = (2 * W_HALF + off + n * fp8_ref.U32) * spread + sub
        # the output's rounding; f16 has subnormals in reach
        room += half * (out.abs() + room) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
        return out, room


def agree(got, out, room, what=""):
    err = (got.double() - out).abs()
    bad = ~(err <= room)
    assert not bad.any(), (what, int(bad.sum()), float((err - room).max()), bad.nonzero()[:4].tolist(),
                           got[bad][:4].tolist(), out[bad][:4].tolist())
