"""Decode attention over FP8 pools with a scale for each token and head,
against 64 bits."""
import math

import pytest
import torch

import tl_attn as tla
from scaled_cache import Pools, agree

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def decode(p, q, partition=0, modulo=False, max_ctx=None, scale=SCALE):
    desc = tla.make_decode_desc(q, p.k, p.tables, p.n_kv, scale, gqa_map=tla.GQA_MODULO if modulo else tla.GQA_GROUPED,
                                partition_tokens=partition, k_scale=float("nan"), v_scale=-1.0)
    ctx = max(p.lens) if max_ctx is None else max_ctx
    ws = torch.full((max(16, tla.workspace_bytes(desc, ctx)),), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, float("nan"))
    tla.paged_attention_decode_scaled(desc, out, q, p.k, p.v, p.ks, p.vs, p.tables, p.lens_dev, ctx, ws)
    torch.cuda.synchronize()
    return out


def check(p, q, out, modulo=False, scale=SCALE, what=""):
    for s, n in enumerate(p.lens):
        want, room = p.attention(q[s:s + 1], s, n, scale, modulo)
        agree(out[s:s + 1], want, room, f"{what} sequence {s} of {n}")


def queries(S, H, dt, seed=1, factor=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (factor * torch.randn(S, H, 128, generator=g, device="cuda")).to(dt)


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 700]


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("BS", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("H,n_kv,modulo", [(32, 8, False), (8, 8, False), (40, 2, True), (16, 1, False), (6, 2, True)])
def test_scaled_decode(BS, dt, H, n_kv, modulo):
    print(f"case scaled decode BS={BS} {dt} {H}/{n_kv} modulo={modulo}", flush=True)
    p = Pools(LENS, n_kv, BS, seed=BS + H)
    q = queries(len(LENS), H, dt)
    check(p, q, decode(p, q, modulo=modulo), modulo)


@pytest.mark.parametrize("BS", [8, 16, 64, 256])
@pytest.mark.parametrize("lens,H,n_kv,partition", [
    ([3000], 32, 8, 0), ([3000], 32, 8, -1), ([5000, 1, 0, 2049], 8, 2, 0), ([2000, 513], 16, 4, 64),
    ([2000, 1999], 16, 4, 192), ([4097, 300], 32, 1, 1024), ([1100] * 20, 32, 8, 0)])
def test_scaled_decode_partitions(BS, lens, H, n_kv, partition):
    print(f"case scaled decode partitions BS={BS} {lens[:4]} {H}/{n_kv} {partition}", flush=True)
    p = Pools(lens, n_kv, BS, seed=3, size=0.8)
    q = queries(len(lens), H, torch.float16)
    check(p, q, decode(p, q, partition))


def test_scaled_decode_partitions_of_a_wavefront():
    """At least 4096 short partitions: a wavefront streams several of them."""
    print("case scaled decode wave partitions", flush=True)
    for BS, lens in ((16, [4100] * 35 + [70, 0]), (8, [4100] * 35 + [700]), (128, [8300] * 17)):
        p = Pools(lens, 8, BS, seed=9, size=0.8)
        q = queries(len(lens), 16, torch.bfloat16)
        out = decode(p, q, 64 if BS != 128 else 128)
        for s in (0, len(lens) // 2, len(lens) - 2, len(lens) - 1):
            want, room = p.attention(q[s:s + 1], s, lens[s], SCALE)
            agree(out[s:s + 1], want, room, f"BS={BS} sequence {s}")


@pytest.mark.parametrize("factor", [2.0 ** -60, 2.0 ** -20, 1.0, 2.0 ** 40])
@pytest.mark.parametrize("size", [0.0, 3.0])
def test_scaled_decode_values_of_any_size(size, factor):
    """Rows whose scales differ by orders of magnitude, and values far outside f16 (bf16 q and out)."""
    print(f"case scaled decode sizes {size} {factor}", flush=True)
    p = Pools([900, 64, 3], 2, 16, seed=4, size=size, v_factor=factor)
    q = queries(3, 8, torch.bfloat16, factor=0.3)
    out = decode(p, q)
    for s, n in enumerate(p.lens):
        want, room = p.attention(q[s:s + 1], s, n, SCALE)
        agree(out[s:s + 1], want, room, f"{size} {factor} sequence {s}")
    assert out.abs().max() > 0


def test_scaled_decode_holes_and_blocks_past_the_pool():
    """Holes, entries past the pool and a row that names nothing; the rows' scales there are NaN or infinite."""
    print("case scaled decode holes", flush=True)
    for BS in (8, 16, 64):
        p = Pools([500, 300, 200, 64], 4, BS, seed=5)
        p.tables[0, 1] = -1
        p.tables[0, p.tables.shape[1] // 3] = p.N
        p.tables[1, 0] = -7
        p.tables[2] = -1
        q = queries(4, 16, torch.float16)
        out = decode(p, q)
        check(p, q, out, what=f"BS={BS}")
        assert not out[2].any()
        # a table narrower than the sequence: the rest is holes
        narrow = p.tables[:, :3].contiguous()
        p.tables = narrow
        check(p, q, decode(p, q), what=f"narrow BS={BS}")


def test_scaled_decode_peaked_and_large_scores():
    """Scores that grow along the sequence: the running maximum is raised again and again, up to weights of 2^8."""
    print("case scaled decode peaked", flush=True)
    p = Pools([1500, 640], 2, 16, seed=6, size=1.0)
    q = queries(2, 8, torch.float16, factor=20.0)
    check(p, q, decode(p, q))
    check(p, q, decode(p, q, partition=256))


def test_scaled_decode_zero_scales_and_nan_rows():
    """Rows kept as zeros count in the sum; a value's NaN scale makes its sequence's heads NaN, a key's leaves them
    unspecified, and no other head is touched."""
    print("case scaled decode zero and nan rows", flush=True)
    p = Pools([200, 100, 70], 2, 16, seed=7)
    for t in (0, 5, 130):
        blk, off = int(p.tables[0, t // 16]), t % 16
        for c, s in ((p.k, p.ks), (p.v, p.vs)):
            c[blk, :, :, off] = 0
            s[blk, :, off] = 0
    p.vs[int(p.tables[1, 2]), 1, 3] = float("nan")
    p.ks[int(p.tables[2, 1]), 0, 4] = float("nan")
    q = queries(3, 8, torch.bfloat16)
    out = decode(p, q)
    want, room = p.attention(q[:1], 0, 200, SCALE)
    agree(out[:1], want, room)
    assert torch.isnan(out[1, 4:]).all() and torch.isfinite(out[1, :4]).all()
    p.ks[int(p.tables[2, 1]), 0, 4] = 0.5
    want, room = p.attention(q[2:], 2, 70, SCALE)
    agree(out[2:, 4:], want[:, 4:], room[:, 4:])


def test_scaled_decode_of_unit_scales_is_the_plain_fp8_decode():
    """With every scale the pool's one scale, the two decodes agree within their rooms."""
    print("case scaled decode unit scales", flush=True)
    p = Pools([333, 1000], 4, 16, seed=8)
    p.ks.fill_(0.01)
    p.vs.fill_(0.02)
    q = queries(2, 16, torch.float16)
    out = decode(p, q)
    desc = tla.make_decode_desc(q, p.k, p.tables, 4, SCALE, k_scale=0.01, v_scale=0.02)
    plain = torch.zeros_like(q)
    ws = torch.empty(max(16, tla.workspace_bytes(desc, 1000)), dtype=torch.uint8, device="cuda")
    tla.paged_attention_decode(desc, plain, q, p.k, p.v, p.tables, p.lens_dev, 1000, ws)
    torch.cuda.synchronize()
    for s, n in enumerate(p.lens):
        want, room = p.attention(q[s:s + 1], s, n, SCALE)
        agree(out[s:s + 1], want, room)
        agree(plain[s:s + 1], want, room)


def test_scaled_decode_far_blocks():
    """A pool past 4 GiB: byte offsets pass 32 bits."""
    print("case scaled decode far blocks", flush=True)
    small = Pools([100, 40], 8, 16, seed=10)
    N = 270000                                              # 4.4 GB a pool
    far = Pools([0], 8, 16)
    far.lens, far.lens_dev, far.N = small.lens, small.lens_dev, N
    far.k, far.v = (torch.empty(N, 8, 128, 16, dtype=torch.uint8, device="cuda") for _ in range(2))
    far.ks, far.vs = (torch.empty(N, 8, 16, device="cuda") for _ in range(2))
    n = small.N
    for name in ("k", "v", "ks", "vs"):
        getattr(far, name)[N - n:] = getattr(small, name)
    far.tables = torch.where(small.tables >= 0, small.tables + (N - n), small.tables)
    q = queries(2, 32, torch.float16)
    assert torch.equal(decode(far, q), decode(small, q))


def test_scaled_decode_replayed_graph():
    print("case scaled decode graph", flush=True)
    p = Pools([2500, 31, 900], 8, 16, seed=11)
    q = queries(3, 32, torch.bfloat16)
    want = decode(p, q)
    desc = tla.make_decode_desc(q, p.k, p.tables, 8, SCALE)
    ws = torch.empty(max(16, tla.workspace_bytes(desc, 2500)), dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tla.paged_attention_decode_scaled(desc, out, q, p.k, p.v, p.ks, p.vs, p.tables, p.lens_dev, 2500, ws)
    for i in range(3):
        out.zero_()
        if i == 2:                                          # the lengths are read at replay
            p.lens_dev.copy_(torch.tensor([1300, 0, 900], dtype=torch.int32))
            p.lens = [1300, 0, 900]
        graph.replay()
        torch.cuda.synchronize()
        if i < 2:
            assert torch.equal(out, want)
        else:
            check(p, q, out)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [[3000], [5, 100, 700]])
def test_scaled_decode_of_a_q_aligned_to_its_elements(dt, lens):
    p = Pools(lens, 8, 16, seed=4)
    q = queries(len(lens), 32, dt)
    odd = torch.empty(q.numel() + 9, dtype=dt, device="cuda")
    for shift in (1, 2, 5):
        view = odd[shift:shift + q.numel()].view(q.shape)
        view.copy_(q)
        check(p, view, decode(p, view), what=f"shift {shift}")
