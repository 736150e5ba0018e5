"""RoPE with several axes on the way into the pools, and the appends that find
a scale for each token and head: bit for bit the oracle's rotation where the
pool has the tensors' type, and within a code's rounding where it is FP8."""
import numpy as np
import pytest
import torch

import fp8_ref
import tl_attn as tla
from test_oracle import rope_tables

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def axis_of_pair(pairs, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(pairs) for _ in range(n)]
    left, got = list(pairs), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                got.append(a)
    return got


def rotated(x, c, s, style):
    """x [T, heads, D] float32 on the CPU; the pair (a, b) becomes (fma(a, c, -fl(b s)), fma(a, s, fl(b c))): the
    fused product is exact in float64, whose sum rounds to float32 as the fused one does but where float64 itself
    lies half way between two float32 values."""
    half = x.shape[2] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if style == tla.ROPE_ADJACENT else (x[..., :half], x[..., half:])
    c, s = c[:, None, :], s[:, None, :]
    r0 = (a.double() * c.double() - (b * s).double()).float()
    r1 = (a.double() * s.double() + (b * c).double()).float()
    return torch.stack((r0, r1), -1).flatten(-2) if style == tla.ROPE_ADJACENT else torch.cat((r0, r1), -1)


class Case:
    """Random tensors of an append.  slots: "runs" (each sequence's tokens in consecutive slots of shuffled blocks,
    from the middle of a block), "steps" (a token per block), "mixed" (any slots)."""

    def __init__(self, T, H, n_kv, D, BS, dt, pairs, interleaved, style, kv="same", slots="runs", seed=0, strided=False):
        g = torch.Generator().manual_seed(seed * 1000 + T + D + BS)
        rng = np.random.default_rng(seed + T)
        self.dims = T, H, n_kv, D, BS
        self.style, self.pairs, self.inter, self.kv = style, pairs, interleaved, kv
        dtype = DT[dt]
        self.max_pos = 4096
        wide = torch.randn(T, (H + 2 * n_kv) * D + (8 if strided else 0), generator=g).to(dtype)
        parts = [wide[:, :H * D], wide[:, H * D:(H + n_kv) * D], wide[:, (H + n_kv) * D:(H + 2 * n_kv) * D]]
        self.q, self.key, self.value = (p.unflatten(1, (n, D)) for p, n in zip(parts, (H, n_kv, n_kv)))
        if strided:
            wide = wide.cuda()
            parts = [wide[:, :H * D], wide[:, H * D:(H + n_kv) * D], wide[:, (H + n_kv) * D:(H + 2 * n_kv) * D]]
            self.dev = [p.unflatten(1, (n, D)) for p, n in zip(parts, (H, n_kv, n_kv))]
        else:
            self.dev = [t.contiguous().cuda() for t in (self.q, self.key, self.value)]
        blocks = T // BS + 3 + (T if slots == "steps" else 0)
        self.N = blocks + 2
        order = rng.permutation(self.N)
        if slots == "runs":
            at = np.arange(T) + BS // 2 + 1
            self.slots = order[at // BS] * BS + at % BS
            if T > 40:
                self.slots[T // 2] = -1                       # a hole in the run
                self.slots[T // 2 + 7] = self.N * BS + 3      # past the pool
        elif slots == "steps":
            self.slots = order[:T] * BS + rng.integers(0, BS, T)
            if T > 3:
                self.slots[2] = -1
            if T > 12:                                        # two tokens in one block
                self.slots[7] = self.slots[5] // BS * BS + (self.slots[5] + 1) % BS
        else:
            self.slots = rng.permutation(self.N * BS)[:T]
        self.slots = torch.from_numpy(self.slots.astype(np.int32))
        self.pos = torch.from_numpy(rng.integers(0, self.max_pos, (len(pairs), T)).astype(np.int32))
        if T > 5:
            self.pos[-1, 4] = self.max_pos                    # off the tables on one axis: not written
            self.pos[0, 5] = -1
        cos, sin = rope_tables(self.max_pos, D)
        self.cos, self.sin = torch.from_numpy(cos), torch.from_numpy(sin)
        shape = (self.N, n_kv, D, BS)
        if kv == "fp8":
            self.k, self.v = (torch.randint(0, 256, shape, generator=g, dtype=torch.uint8) for _ in range(2))
            self.ks, self.vs = (torch.randn(self.N, n_kv, BS, generator=g) for _ in range(2))
        else:
            self.k, self.v = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
            self.ks = self.vs = None

    def call(self, q_out=None, q=None):
        up = [t if t is None else t.cuda() for t in (self.k, self.v, self.ks, self.vs)]
        k, v, ks, vs = up
        q = self.dev[0] if q is None else q
        desc = tla.make_rope_axes_desc(q, self.dev[1], k, self.pairs, self.max_pos, style=self.style,
                                       interleaved=self.inter)
        tla.rope_axes_reshape_and_cache(desc, q, self.dev[1], self.dev[2], k, v, self.slots.cuda(), self.pos.cuda(),
                                        self.cos.cuda(), self.sin.cuda(), q_out=q_out, k_scales=ks, v_scales=vs)
        torch.cuda.synchronize()
        return up

    def reference(self):
        T, H, n_kv, D, BS = self.dims
        there = ((self.pos >= 0) & (self.pos < self.max_pos)).all(0)
        axis = torch.tensor(axis_of_pair(self.pairs, self.inter))
        rows = self.pos.clamp(0, self.max_pos - 1).long()[axis].t()
        c, s = (t[rows, torch.arange(D // 2)] for t in (self.cos, self.sin))
        written = there & (self.slots >= 0) & (self.slots < self.N * BS)
        return (there, written, rotated(self.q.float(), c, s, self.style), rotated(self.key.float(), c, s, self.style))

    def check(self, got, q_out, q_before):
        T, H, n_kv, D, BS = self.dims
        there, written, q_ref, k_ref = self.reference()
        want = q_before.cpu().clone()
        want[there] = q_ref[there].to(want.dtype)
        assert torch.equal(q_out.cpu(), want)
        s = self.slots.long()[written]
        blk, off = s // BS, s % BS
        k, v, ks, vs = (t if t is None else t.cpu() for t in got)
        rows = {"k": k_ref[written], "v": self.value.float()[written]}
        for name, pool, before, scales, scales0 in (("k", k, self.k, ks, self.ks), ("v", v, self.v, vs, self.vs)):
            rest = before.clone()
            if scales is None:
                rest[blk, :, :, off] = rows[name].to(rest.dtype)
                assert torch.equal(pool.view(torch.uint8), rest.view(torch.uint8)), name
                continue
            # the row is exact but for the fused product's half-way cases: one rounding of fp32
            fp8_ref.check(pool[blk, :, :, off], scales[blk, :, off], rows[name].double(), fp8_ref.U32, name)
            rest[blk, :, :, off] = pool[blk, :, :, off]
            assert torch.equal(pool, rest), name               # every other code is as it was
            rest = scales0.clone()
            rest[blk, :, off] = scales[blk, :, off]
            assert torch.equal(scales, rest), name


AXES = {128: [([64], False), ([16, 24, 24], False), ([24, 20, 20], True), ([21, 21, 22], False), ([5, 0, 50, 9], True)],
        64: [([32], False), ([8, 12, 12], True)], 96: [([3, 45], False)], 256: [([40, 44, 44], True)], 80: [([40], False)]}


@pytest.mark.parametrize("style", [tla.ROPE_ADJACENT, tla.ROPE_HALVES])
@pytest.mark.parametrize("dt,kv", [("f16", "same"), ("bf16", "same"), ("f32", "same"), ("f16", "fp8"), ("bf16", "fp8")])
@pytest.mark.parametrize("T,H,n_kv,D,BS,slots", [
    (1, 32, 8, 128, 16, "steps"), (64, 32, 8, 128, 16, "steps"), (33, 8, 2, 128, 32, "steps"), (20, 4, 4, 128, 8, "steps"),
    (9, 16, 2, 128, 64, "steps"), (7, 8, 8, 128, 256, "steps"), (13, 5, 3, 128, 20, "steps"), (300, 8, 2, 128, 16, "steps"),
    (50, 8, 2, 128, 16, "runs"), (256, 32, 8, 128, 16, "runs"), (257, 8, 2, 128, 8, "runs"), (700, 32, 8, 128, 16, "runs"),
    (601, 64, 8, 128, 32, "runs"), (530, 8, 1, 128, 64, "runs"), (900, 4, 4, 128, 256, "runs"), (400, 6, 2, 128, 24, "runs"),
    (350, 8, 2, 128, 16, "mixed"), (90, 0, 4, 128, 16, "runs"),
    (40, 8, 2, 64, 16, "steps"), (450, 8, 2, 64, 16, "runs"), (300, 4, 2, 96, 16, "runs"), (300, 4, 2, 256, 16, "runs"),
    (21, 4, 2, 256, 16, "steps"), (300, 4, 4, 80, 16, "mixed")])
def test_rope_axes_append(style, dt, kv, T, H, n_kv, D, BS, slots):
    if kv == "fp8" and D != 128:
        pytest.skip("scaled FP8 pools have head size 128")
    choice = AXES[D]
    pairs, inter = choice[(T + style) % len(choice)]
    print(f"case axes T={T} H={H} n_kv={n_kv} D={D} BS={BS} {dt} {kv} {slots} {pairs} {inter} {style}", flush=True)
    c = Case(T, H, n_kv, D, BS, dt, pairs, inter, style, kv, slots, seed=style)
    if H == 0:
        c.dev[0] = c.q = torch.zeros(T, 0, D, dtype=DT[dt])
        k, v = c.k.cuda(), c.v.cuda()
        ks, vs = (None, None) if c.ks is None else (c.ks.cuda(), c.vs.cuda())
        desc = tla.make_rope_axes_desc(None, c.dev[1], k, pairs, c.max_pos, style=style, interleaved=inter)
        tla.rope_axes_reshape_and_cache(desc, None, c.dev[1], c.dev[2], k, v, c.slots.cuda(), c.pos.cuda(), c.cos.cuda(),
                                        c.sin.cuda(), k_scales=ks, v_scales=vs)
        torch.cuda.synchronize()
        c.check((k, v, ks, vs), c.q, c.q)
        return
    q_out = torch.full_like(c.dev[0], 3.0)
    before = q_out.clone()
    c.check(c.call(q_out), q_out, before)


@pytest.mark.parametrize("kv", ["same", "fp8"])
@pytest.mark.parametrize("T,slots", [(17, "steps"), (100, "runs"), (610, "runs")])
def test_rope_axes_slices_of_one_projection_in_place(kv, T, slots):
    """q, key and value are slices of one tensor, the tokens' strides wider than their heads; q is turned in place."""
    c = Case(T, 8, 2, 128, 16, "bf16", [24, 20, 20], True, tla.ROPE_HALVES, kv, slots, strided=True)
    print(f"case axes strided T={T} {kv}", flush=True)
    before = c.dev[0].clone()
    key, value = c.dev[1].clone(), c.dev[2].clone()
    got = c.call()
    c.check(got, c.dev[0], before)
    assert torch.equal(key, c.dev[1]) and torch.equal(value, c.dev[2])


@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("kv", ["same", "fp8"])
@pytest.mark.parametrize("T,slots", [(17, "steps"), (610, "runs")])
def test_rope_axes_unaligned_tensors(T, slots, kv, shift):
    """Tensors (and 2-byte pools) that begin `shift` elements past an aligned address."""
    c = Case(T, 8, 2, 128, 16, "f16", [16, 24, 24], False, tla.ROPE_ADJACENT, kv, slots)

    def moved(t):
        if t is None:
            return None
        flat = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")
        flat[shift:] = t.cuda().flatten()
        return flat[shift:].view(t.shape)
    print(f"case axes unaligned T={T} {kv} shift={shift}", flush=True)
    q, key, value, k, v, ks, vs = (moved(t) for t in (c.q, c.key, c.value, c.k, c.v, c.ks, c.vs))
    cos, sin, slots_d, pos = moved(c.cos), moved(c.sin), moved(c.slots), moved(c.pos)
    q_out = moved(torch.zeros(c.q.shape, dtype=c.q.dtype))
    desc = tla.make_rope_axes_desc(q, key, k, c.pairs, c.max_pos, style=c.style)
    tla.rope_axes_reshape_and_cache(desc, q, key, value, k, v, slots_d, pos, cos, sin, q_out=q_out, k_scales=ks,
                                    v_scales=vs)
    torch.cuda.synchronize()
    c.check((k, v, ks, vs), q_out, torch.zeros_like(c.q))


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("T,slots", [(40, "steps"), (700, "runs")])
def test_one_axis_is_the_plain_rope_append(dt, T, slots):
    c = Case(T, 32, 8, 128, 16, dt, [64], False, tla.ROPE_ADJACENT, "same", slots)
    print(f"case axes one axis T={T} {dt}", flush=True)
    a, b = torch.zeros_like(c.dev[0]), torch.zeros_like(c.dev[0])
    k, v, _, _ = c.call(a)
    k2, v2 = c.k.cuda(), c.v.cuda()
    tla.rope_reshape_and_cache(c.dev[0], c.dev[1], c.dev[2], k2, v2, c.slots.cuda(), c.pos[0].contiguous().cuda(),
                               c.cos.cuda(), c.sin.cuda(), c.style, q_out=b)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(k, k2) and torch.equal(v, v2)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("T,n_kv,BS,slots", [(1, 8, 16, "steps"), (64, 8, 16, "steps"), (19, 3, 64, "steps"),
                                             (11, 2, 256, "steps"), (300, 8, 32, "steps"), (200, 8, 16, "runs"),
                                             (900, 8, 16, "runs"), (513, 1, 8, "runs"), (300, 2, 12, "mixed")])
def test_reshape_and_cache_fp8_scaled(dt, T, n_kv, BS, slots):
    c = Case(T, 1, n_kv, 128, BS, dt, [64], False, 0, "fp8", slots)
    c.pos.clamp_(0, c.max_pos - 1)
    up = [t.cuda() for t in (c.k, c.v, c.ks, c.vs)]
    print(f"case fp8 scaled append T={T} n_kv={n_kv} BS={BS} {dt} {slots}", flush=True)
    tla.reshape_and_cache_fp8_scaled(c.dev[1], c.dev[2], *up, c.slots.cuda())
    torch.cuda.synchronize()
    c.reference = lambda: (torch.ones(T, dtype=torch.bool), (c.slots >= 0) & (c.slots < c.N * BS), c.q.float(),
                           c.key.float())
    c.check(up, c.q, c.q)


@pytest.mark.parametrize("T,slots", [(12, "steps"), (300, "runs")])
def test_scaled_rows_of_zeros_infinities_and_nan(T, slots):
    """A row of zeros reads as zeros, one with an infinity or a NaN as NaN, and no other row does."""
    c = Case(T, 1, 2, 128, 16, "bf16", [64], False, 0, "fp8", slots)
    key, value = c.dev[1], c.dev[2]
    key[0, 0] = 0
    key[1, 1, 77] = float("nan")
    value[1, 0, 3] = float("-inf")
    value[3, 1] = 1e-38                                     # below 448 x 2^-126
    up = [t.cuda() for t in (c.k, c.v, c.ks, c.vs)]
    print(f"case fp8 scaled special T={T}", flush=True)
    tla.reshape_and_cache_fp8_scaled(key, value, *up, c.slots.cuda())
    torch.cuda.synchronize()
    k, v, ks, vs = (t.cpu() for t in up)
    s = c.slots.long()

    def read(pool, scales, t, h):
        blk, off = s[t] // 16, s[t] % 16
        return fp8_ref.values(pool[blk, h, :, off]) * scales[blk, h, off].double()
    assert not read(k, ks, 0, 0).any() and not read(v, vs, 3, 1).any()
    assert torch.isnan(read(k, ks, 1, 1)).all() and torch.isnan(read(v, vs, 1, 0)).all()
    for pool, scales, t, h, rows in ((k, ks, 1, 0, key), (v, vs, 1, 1, value), (k, ks, 4, 1, key), (v, vs, 3, 0, value)):
        x = rows[t, h].cpu().double()
        assert (read(pool, scales, t, h) - x).abs().max() <= fp8_ref.CODE * x.abs().max()


@pytest.mark.parametrize("kv", ["same", "fp8"])
@pytest.mark.parametrize("T,slots", [(48, "steps"), (700, "runs")])
def test_rope_axes_replayed_graph_and_another_stream(kv, T, slots):
    c = Case(T, 32, 8, 128, 16, "bf16", [16, 24, 24], False, tla.ROPE_HALVES, kv, slots)
    a = torch.zeros_like(c.dev[0])
    print(f"case axes graph {kv} T={T}", flush=True)
    want = c.call(a)
    first = [t if t is None else t.cuda() for t in (c.k, c.v, c.ks, c.vs)]
    k, v, ks, vs = (t if t is None else t.clone() for t in first)
    b = torch.zeros_like(a)
    desc = tla.make_rope_axes_desc(c.dev[0], c.dev[1], k, c.pairs, c.max_pos, style=c.style)
    slots_d, pos, cos, sin = c.slots.cuda(), c.pos.cuda(), c.cos.cuda(), c.sin.cuda()

    def step():
        tla.rope_axes_reshape_and_cache(desc, c.dev[0], c.dev[1], c.dev[2], k, v, slots_d, pos, cos, sin, q_out=b,
                                        k_scales=ks, v_scales=vs)

    def same():
        torch.cuda.synchronize()
        assert torch.equal(a, b)
        for x, y in zip(want, (k, v, ks, vs)):
            assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))

    def again():
        b.zero_()
        for x, y in zip((k, v, ks, vs), first):
            if x is not None:
                x.copy_(y)
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    same()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        again()
        graph.replay()
        same()


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_the_scale_of_every_magnitude(dt):
    """A row of one magnitude for each positive finite value: scale a / 448 to the bit, as fp32 divides, and the code
    of 448 (0x7E) or, negative, of -448; below 448 x 2^-126 the scale 0 and zeros."""
    n = 0x7C00 if dt == torch.float16 else 0x7F80
    a = torch.arange(n, dtype=torch.int16).view(dt)
    want = a.float() / 448
    want[want < 2.0 ** -126] = 0
    key = a.view(n, 1, 1).expand(n, 1, 128).contiguous().cuda()
    BS, N = 16, (n + 15) // 16
    k, v = (torch.full((N, 1, 128, BS), 0x55, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((N, 1, BS), -1.0, device="cuda") for _ in range(2))
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    for part in (slice(0, n), slice(5, 300)):                # tiles, and a step
        tla.reshape_and_cache_fp8_scaled(key[part], -key[part], k, v, ks, vs, slots[part])
        torch.cuda.synchronize()
        for scales, codes, sign in ((ks, k, 0), (vs, v, 0x80)):
            assert torch.equal(scales.view(-1)[part].cpu(), want[part])
            rows = codes.permute(0, 3, 1, 2).reshape(-1, 128)[part].cpu()
            live = want[part] > 0
            assert (rows[live] == 0x7E | sign).all() and ((rows[~live] & 0x7F) == 0).all()
        ks.fill_(-1.0), vs.fill_(-1.0), k.fill_(0x55), v.fill_(0x55)
