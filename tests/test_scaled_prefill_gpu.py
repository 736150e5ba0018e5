"""Chunk attention (with decode rows beside it) over FP8 pools with a scale for
each token and head, against 64 bits; and the 8-bit step as a whole."""
import math

import pytest
import torch

import fp8_ref
import tl_attn as tla
from scaled_cache import Pools, agree

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def chunk(p, q, q_lens, modulo=False, prompts=0, stream=None):
    cu = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)), dtype=torch.int32, device="cuda")
    desc = tla.make_prefill_desc(q, p.k, p.tables, len(p.lens), p.n_kv, SCALE, num_prefill_seqs=prompts,
                                 gqa_map=tla.GQA_MODULO if modulo else tla.GQA_GROUPED, kv_dtype=tla.FP8_E4M3,
                                 k_scale=-1.0, v_scale=float("nan"))
    out = torch.full_like(q, 7.0)
    tla.chunked_prefill_scaled(desc, out, q, cu, p.k, p.v, p.ks, p.vs, p.tables, p.lens_dev, max(q_lens))
    torch.cuda.synchronize()
    return out


def check(p, q, q_lens, out, modulo=False, what=""):
    at = 0
    for s, (n, L) in enumerate(zip(q_lens, p.lens)):
        if n:
            want, room = p.attention(q[at:at + n], s, L, SCALE, modulo)
            agree(out[at:at + n], want, room, f"{what} sequence {s}: {n} of {L}")
        at += n
    assert (out[at:] == 7.0).all()                          # rows behind the last sequence are left as they were


def queries(T, H, dt, seed=1, factor=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (factor * torch.randn(T, H, 128, generator=g, device="cuda")).to(dt)


# few tiles (the keys split over a workgroup's wavefronts), with decode rows and an empty chunk
SMALL = [(2, 2), (5, 5), (64, 64), (17, 130), (1, 77), (0, 40), (100, 301), (1, 1)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("BS", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("H,n_kv,modulo", [(8, 2, False), (6, 2, True), (5, 5, False)])
def test_scaled_chunks(BS, dt, H, n_kv, modulo):
    print(f"case scaled chunks BS={BS} {dt} {H}/{n_kv} {modulo}", flush=True)
    q_lens = [n for n, _ in SMALL]
    p = Pools([L for _, L in SMALL], n_kv, BS, seed=BS + H, size=0.7)
    q = queries(sum(q_lens) + 3, H, dt)
    check(p, q, q_lens, chunk(p, q, q_lens, modulo), modulo)


# many tiles (two groups of wavefronts in turn)
LARGE = [(300, 300), (257, 700), (64, 1000), (511, 513)]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("BS", [8, 16, 32, 64, 128, 256])
def test_scaled_chunks_of_many_tiles(BS, dt):
    print(f"case scaled large chunks BS={BS} {dt}", flush=True)
    q_lens = [n for n, _ in LARGE] + [1, 1]
    p = Pools([L for _, L in LARGE] + [900, 64], 8, BS, seed=BS, size=0.7)
    q = queries(sum(q_lens), 32, dt)
    check(p, q, q_lens, chunk(p, q, q_lens, prompts=len(LARGE)))


@pytest.mark.parametrize("tiles", ["few", "many"])
@pytest.mark.parametrize("dt,factor,size", [
    (torch.float16, 2.0 ** -12, 1.0), (torch.float16, 100.0, 0.5), (torch.bfloat16, 2.0 ** -60, 1.0),
    (torch.bfloat16, 1.0, 3.0), (torch.bfloat16, 2.0 ** 40, 1.0)])
def test_scaled_chunks_values_of_any_size(tiles, dt, factor, size):
    """Values far outside f16 with bf16 out, and rows whose scales differ by orders of magnitude."""
    print(f"case scaled chunk sizes {tiles} {dt} {factor} {size}", flush=True)
    rows = [(40, 500)] if tiles == "few" else [(300, 600)]
    n_kv, H = (2, 8) if tiles == "few" else (32, 64)
    p = Pools([L for _, L in rows], n_kv, 16, seed=3, size=size, v_factor=factor)
    q_lens = [n for n, _ in rows]
    q = queries(sum(q_lens), H, dt, factor=0.3)
    out = chunk(p, q, q_lens)
    check(p, q, q_lens, out)
    assert out.abs().max() > 0


@pytest.mark.parametrize("tiles", ["few", "many"])
def test_scaled_chunks_values_that_grow_along_the_sequence(tiles):
    """The value scales' unit is raised again and again, in rows of zeros' company."""
    print(f"case scaled chunk growing values {tiles}", flush=True)
    rows, n_kv, H = ([(40, 500)], 2, 8) if tiles == "few" else ([(300, 600)], 32, 64)
    p = Pools([L for _, L in rows], n_kv, 16, seed=4)
    for b in range((rows[0][1] + 15) // 16):
        blk = int(p.tables[0, b])
        p.vs[blk] *= 2.0 ** (b / 2 - 10)
    zero = int(p.tables[0, 0])
    p.v[zero], p.vs[zero] = 0, 0
    q = queries(rows[0][0], H, torch.bfloat16)
    check(p, q, [rows[0][0]], chunk(p, q, [rows[0][0]]))


def test_scaled_chunks_holes():
    print("case scaled chunk holes", flush=True)
    for BS, H, n_kv, rows in ((16, 8, 2, [(40, 300), (30, 100), (20, 64)]), (8, 8, 2, [(40, 300), (30, 100), (20, 64)]),
                              (32, 64, 8, [(200, 900), (256, 300), (300, 300)])):
        p = Pools([L for _, L in rows], n_kv, BS, seed=5)
        p.tables[0, 1] = -1
        p.tables[0, 4] = p.N + 9
        p.tables[1, 0] = -1
        p.tables[2] = -1                                    # nothing left to attend to
        q_lens = [n for n, _ in rows]
        q = queries(sum(q_lens), H, torch.float16)
        out = chunk(p, q, q_lens)
        check(p, q, q_lens, out, what=f"BS={BS}")
        assert not out[q_lens[0] + q_lens[1]:].any()


def test_scaled_chunks_peaked_scores():
    print("case scaled chunk peaked", flush=True)
    for H, n_kv, rows in ((8, 2, [(60, 500)]), (64, 8, [(400, 900)])):
        p = Pools([L for _, L in rows], n_kv, 16, seed=6, size=1.0)
        q_lens = [n for n, _ in rows]
        q = queries(sum(q_lens), H, torch.bfloat16, factor=15.0)
        check(p, q, q_lens, chunk(p, q, q_lens))


def test_scaled_chunk_replayed_graph_and_another_stream():
    print("case scaled chunk graph", flush=True)
    p = Pools([600, 500, 70], 8, 16, seed=8)
    q_lens = [300, 200, 1]
    q = queries(501, 32, torch.bfloat16)
    want = chunk(p, q, q_lens)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(chunk(p, q, q_lens), want)
    cu = torch.tensor([0, 300, 500, 501], dtype=torch.int32, device="cuda")
    desc = tla.make_prefill_desc(q, p.k, p.tables, 3, 8, SCALE, kv_dtype=tla.FP8_E4M3)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tla.chunked_prefill_scaled(desc, out, q, cu, p.k, p.v, p.ks, p.vs, p.tables, p.lens_dev, 300)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("BS", [16, 64])
def test_the_step_as_a_whole(dt, BS):
    """A layer as a server runs it: norm to FP8 codes, the projection of what they stand for, rotation on three axes
    into the scaled pools, chunk attention; then a token more for each sequence and its decode.  Each operator is
    compared with 64 bits on what the one before it left."""
    print(f"case 8-bit step {dt} BS={BS}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(2)
    hidden, H, n_kv, D = 512, 8, 2, 128
    prompts = [200, 33, 90]
    T, S = sum(prompts), len(prompts)
    counts = [(n + 1 + BS - 1) // BS for n in prompts]
    N = sum(counts) + 3
    order = torch.randperm(N, generator=g, device="cuda").to(torch.int32)
    p = Pools([0] * S, n_kv, BS, extra_blocks=N, max_blocks=max(counts))
    for s, n in enumerate(counts):
        p.tables[s, :n] = order[sum(counts[:s]):sum(counts[:s]) + n]
    weight = (1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(dt)
    w_qkv = torch.randn(hidden, (H + 2 * n_kv) * D, generator=g, device="cuda") / math.sqrt(hidden)
    ang = torch.outer(torch.arange(512, dtype=torch.float64),
                      10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    cos, sin = ang.cos().float().cuda(), ang.sin().float().cuda()
    pairs = [16, 24, 24]
    axis = torch.tensor([a for a, n in enumerate(pairs) for _ in range(n)], device="cuda")

    def layer(x, res, pos, slots):
        rows = x.shape[0]
        codes = torch.empty(rows, hidden, dtype=torch.uint8, device="cuda")
        scales = torch.empty(rows, hidden // 128, device="cuda")
        tla.fused_add_rms_norm_fp8(codes, scales, res, x, weight, 1e-5, 128)
        value = (fp8_ref.values(codes).view(rows, -1, 128) * scales.double()[..., None]).view(rows, hidden)
        r = res.double()
        want = r / torch.sqrt((r * r).mean(1, keepdim=True) + 1e-5) * weight.double()
        # the residual as stored is off by its rounding in the sum of squares only
        assert ((value - want).abs() <= (2.0 ** -4 + 2.0 ** -7) * want.abs() + 2.0 ** -10 * scales.amax()).all()
        qkv = (value.float() @ w_qkv).to(dt)
        q, key, val = qkv.split([H * D, n_kv * D, n_kv * D], 1)
        q, key, val = q.unflatten(1, (H, D)), key.unflatten(1, (n_kv, D)), val.unflatten(1, (n_kv, D))
        turned = torch.empty(rows, H, D, dtype=dt, device="cuda")
        desc = tla.make_rope_axes_desc(q, key, p.k, pairs, 512, style=tla.ROPE_HALVES)
        tla.rope_axes_reshape_and_cache(desc, q, key, val, p.k, p.v, slots, pos, cos, sin, q_out=turned,
                                        k_scales=p.ks, v_scales=p.vs)
        at = pos.long()[axis].t()
        c, sn = (t.double()[at, torch.arange(64, device="cuda")][:, None, :] for t in (cos, sin))

        def turn(x):
            a, b = x.double().chunk(2, -1)
            return torch.cat((a * c - b * sn, a * sn + b * c), -1)
        half = 2.0 ** -11 if dt == torch.float16 else 2.0 ** -8
        size = q.double().abs()
        size = (size + size.roll(64, -1)) * 2.0 ** -22
        assert ((turned.double() - turn(q)).abs() <= half * turn(q).abs() + size + 2.0 ** -24).all()
        blk, off = slots.long() // BS, slots.long() % BS
        k_ref = turn(key)
        # two products and a sum in fp32: relative to the pair, not to the result
        top = k_ref.abs().amax(-1)
        got = fp8_ref.values(p.k[blk, :, :, off]) * p.ks[blk, :, off].double()[..., None]
        assert ((got - k_ref).abs() <= fp8_ref.CODE * k_ref.abs() + 2.0 ** -18 * top[..., None]).all()
        fp8_ref.check(p.v[blk, :, :, off], p.vs[blk, :, off], val.double(), 0.0, "values")
        return turned

    def places(first, counts_of):
        pos, slots = [], []
        for s, n in enumerate(counts_of):
            t = torch.arange(first[s], first[s] + n, device="cuda")
            pos.append(torch.stack([t, t // 3, t % 7]))
            slots.append(p.tables[s, t // BS] * BS + (t % BS).int())
        return torch.cat(pos, 1).int().contiguous(), torch.cat(slots).int()

    x = torch.randn(T, hidden, generator=g, device="cuda").to(dt)
    res = torch.randn(T, hidden, generator=g, device="cuda").to(dt)
    pos, slots = places([0] * S, prompts)
    q = layer(x, res, pos, slots)
    p.lens, p.lens_dev = prompts, torch.tensor(prompts, dtype=torch.int32, device="cuda")
    check(p, q, prompts, chunk(p, q, prompts), what="prompts")
    x = torch.randn(S, hidden, generator=g, device="cuda").to(dt)
    res = torch.randn(S, hidden, generator=g, device="cuda").to(dt)
    pos, slots = places(prompts, [1] * S)
    before = p.k.clone()
    q = layer(x, res, pos, slots)
    changed = (p.k != before).any(dim=2)                    # [N, n_kv, BS]
    changed[slots.long() // BS, :, slots.long() % BS] = False
    assert not changed.any()
    p.lens = [n + 1 for n in prompts]
    p.lens_dev = torch.tensor(p.lens, dtype=torch.int32, device="cuda")
    desc = tla.make_decode_desc(q, p.k, p.tables, n_kv, SCALE)
    out = torch.empty_like(q)
    ws = torch.empty(max(16, tla.workspace_bytes(desc, max(p.lens))), dtype=torch.uint8, device="cuda")
    tla.paged_attention_decode_scaled(desc, out, q, p.k, p.v, p.ks, p.vs, p.tables, p.lens_dev, max(p.lens), ws)
    torch.cuda.synchronize()
    for s, n in enumerate(p.lens):
        want, room = p.attention(q[s:s + 1], s, n, SCALE)
        agree(out[s:s + 1], want, room, f"step, sequence {s}")
    # blocks move with their scales
    mapping = torch.tensor([[int(p.tables[0, 0]), N - 1 if int(p.tables[0, 0]) != N - 1 else 0]], dtype=torch.int32,
                           device="cuda")
    src, dst = mapping[0].tolist()
    if dst not in p.tables.tolist()[0]:
        tla.copy_blocks(p.k, p.v, mapping)
        tla.copy_blocks(p.ks, p.vs, mapping)
        p.tables[0, 0] = dst
        again = torch.empty_like(out)
        tla.paged_attention_decode_scaled(desc, again, q, p.k, p.v, p.ks, p.vs, p.tables, p.lens_dev, max(p.lens), ws)
        torch.cuda.synchronize()
        assert torch.equal(again[0], out[0])
