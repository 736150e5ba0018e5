"""RMSNorm and residual add + RMSNorm with FP8 codes and scales, against the
same in 64 bits."""
import pytest
import torch

import fp8_ref
import tl_attn as tla

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _off(hidden):
    """Relative error of the norm's fp32 result before it is rounded to a code.  The sum of H squares: each square
    and each addition is off by half a step; a thread adds at most H / 64 of them in turn and 8 levels of lanes and
    wavefronts follow.  The root halves that.  Then mean, eps, root, reciprocal and two products: 6 roundings."""
    return ((hidden / 64 + 10) / 2 + 6) * fp8_ref.U32


def _reference(x, w, eps, res=None):
    """(y in float64, the residual as stored) from the definition."""
    dt = x.dtype
    r = x.double()
    kept = None
    if res is not None:
        r32 = x.float() + res.float()
        kept = r32.to(dt)
        r = r32.double()
    inv = 1.0 / torch.sqrt((r * r).mean(-1, keepdim=True) + eps)
    return (kept.double() if res is not None else r) * inv * w.double(), kept


def _run(T, H, dt, group, fused, g, eps=1e-5):
    x = (3 * torch.randn(T, H, generator=g, device="cuda")).to(DT[dt])
    res = torch.randn(T, H, generator=g, device="cuda").to(DT[dt])
    w = (1 + 0.2 * torch.randn(H, generator=g, device="cuda")).to(DT[dt])
    out = torch.full((T, H), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((T, H // group) if group else (T,), -1.0, device="cuda")
    want, kept = _reference(x, w, eps, res if fused else None)
    if fused:
        tla.fused_add_rms_norm_fp8(out, scales, res, x, w, eps, group)
    else:
        tla.rms_norm_fp8(out, scales, x, w, eps, group)
    torch.cuda.synchronize()
    if fused:
        assert torch.equal(res, kept)                       # the residual's update is exact
    rows = want.view(T, H // group, group) if group else want
    fp8_ref.check(out.view(rows.shape), scales, rows, _off(H), f"T={T} H={H} {dt} group={group}")


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("T,H,group", [
    (1, 8, 0), (1, 1, 0), (3, 96, 32), (5, 100, 0), (7, 64, 64), (64, 4096, 0), (64, 4096, 128), (2, 512, 256),
    (33, 1024, 64), (17, 5632, 0), (17, 5632, 256), (9, 1032, 0), (4, 8192, 32), (3, 14336, 128), (3, 14336, 0),
    (2, 16384, 0), (2, 16392, 0), (2, 28672, 256), (1, 40000, 64), (300, 2048, 128)])
def test_norm_fp8(T, H, group, dt, fused):
    g = torch.Generator(device="cuda").manual_seed(T * 7 + H + group)
    print(f"case norm_fp8 T={T} H={H} group={group} {dt} fused={fused}", flush=True)
    _run(T, H, dt, group, fused, g)


@pytest.mark.parametrize("dt", ["f16", "f32"])
@pytest.mark.parametrize("group", [0, 32])
def test_norm_fp8_unaligned_rows(dt, group):
    """Tensors that begin one element past an aligned address, rows of an odd number of elements."""
    g = torch.Generator(device="cuda").manual_seed(5)
    H = 96 if group else 101
    x = torch.randn(3 * H + 1, generator=g, device="cuda").to(DT[dt])[1:].view(3, H)
    w = torch.randn(H + 1, generator=g, device="cuda").to(DT[dt])[1:]
    res = torch.randn(3 * H + 1, generator=g, device="cuda").to(DT[dt])[1:].view(3, H)
    want, kept = _reference(x, w, 1e-6, res)
    out = torch.zeros(3 * H + 1, dtype=torch.uint8, device="cuda")[1:].view(3, H)
    scales = torch.zeros((3, H // group) if group else (3,), device="cuda")
    print(f"case norm_fp8 unaligned {dt} group={group}", flush=True)
    tla.fused_add_rms_norm_fp8(out, scales, res, x, w, 1e-6, group)
    torch.cuda.synchronize()
    assert torch.equal(res, kept)
    rows = want.view(3, H // group, group) if group else want
    fp8_ref.check(out.view(rows.shape), scales, rows, _off(H))


@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("H", [512, 4096, 4100])
def test_norm_fp8_zero_infinite_and_nan_rows(H, group):
    """A row of zeros is kept as zeros under scale 0; an infinity or a NaN makes its row (its group, where the others
    stay finite only if the norm does) read as NaN, and no other row."""
    if group and H % group:
        pytest.skip("no whole groups")
    x = torch.randn(5, H, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    x[1] = 0
    x[2, H // 2] = float("nan")
    x[3, 3] = float("inf")
    w = torch.ones(H, dtype=torch.float16, device="cuda")
    out = torch.zeros(5, H, dtype=torch.uint8, device="cuda")
    scales = torch.zeros((5, H // group) if group else (5,), device="cuda")
    print(f"case norm_fp8 special H={H} group={group}", flush=True)
    tla.rms_norm_fp8(out, scales, x, w, 1e-5, group)
    torch.cuda.synchronize()
    s = scales.view(5, -1)
    assert not s[1].any() and not fp8_ref.values(out[1]).any()
    read = fp8_ref.values(out).view(5, s.shape[1], -1) * s.double()[..., None]
    assert torch.isnan(read[2]).all()                       # the sum of squares is NaN
    assert torch.isnan(read[3].flatten()[3])                # inf * 0
    assert torch.isfinite(read[[0, 4]]).all()
    want, _ = _reference(x[[0, 4]], w, 1e-5)
    rows = want.view(2, -1, group) if group else want
    fp8_ref.check(out[[0, 4]].view(rows.shape), scales[[0, 4]], rows, _off(H))


def test_norm_fp8_equals_itself_in_a_replayed_graph_and_on_another_stream():
    T, H = 37, 4096
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    res0 = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    w = torch.randn(H, generator=g, device="cuda").bfloat16()

    def fresh():
        return torch.zeros(T, H, dtype=torch.uint8, device="cuda"), torch.zeros(T, H // 128, device="cuda"), res0.clone()
    a, b = fresh(), fresh()
    print("case norm_fp8 graph", flush=True)
    tla.fused_add_rms_norm_fp8(a[0], a[1], a[2], x, w, 1e-5, 128)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    c = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tla.fused_add_rms_norm_fp8(c[0], c[1], c[2], x, w, 1e-5, 128)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tla.fused_add_rms_norm_fp8(b[0], b[1], b[2], x, w, 1e-5, 128)
    for _ in range(3):
        b[0].zero_()
        b[1].zero_()
        b[2].copy_(res0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
