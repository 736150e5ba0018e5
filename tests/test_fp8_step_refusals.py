"""The 8-bit step's entry points refuse what they do not take, before any HIP
call: no GPU needed."""
import ctypes

import pytest
import torch

import tl_attn as tla

FAKE = ctypes.c_void_p(0x1000)          # never dereferenced: every call below is refused or has no work
ODD = ctypes.c_void_p(0x1001)
L = tla.lib


def _norm(T=4, H=256, group=0, dtype=tla.BF16, out=FAKE, scales=FAKE, x=FAKE, w=FAKE, res=FAKE, fused=True):
    if fused:
        return L.tl_fused_add_rms_norm_fp8(out, scales, res, x, w, T, H, group, 1e-5, dtype, None)
    return L.tl_rms_norm_fp8(out, scales, x, w, T, H, group, 1e-5, dtype, None)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), tla.ERR_INVALID_ARGUMENT), (dict(H=0), tla.ERR_INVALID_ARGUMENT),
    (dict(dtype=tla.FP8_E4M3), tla.ERR_INVALID_ARGUMENT), (dict(dtype=7), tla.ERR_INVALID_ARGUMENT),
    (dict(group=48), tla.ERR_NOT_IMPLEMENTED), (dict(group=-32), tla.ERR_NOT_IMPLEMENTED),
    (dict(group=512, H=512), tla.ERR_NOT_IMPLEMENTED), (dict(group=128, H=200), tla.ERR_INVALID_ARGUMENT),
    (dict(out=None), tla.ERR_INVALID_ARGUMENT), (dict(scales=None), tla.ERR_INVALID_ARGUMENT),
    (dict(x=None), tla.ERR_INVALID_ARGUMENT), (dict(w=None), tla.ERR_INVALID_ARGUMENT),
    (dict(x=ODD), tla.ERR_INVALID_ARGUMENT), (dict(w=ODD), tla.ERR_INVALID_ARGUMENT),
    (dict(scales=ctypes.c_void_p(0x1002)), tla.ERR_INVALID_ARGUMENT),
    (dict(x=ctypes.c_void_p(0x1002), dtype=tla.F32), tla.ERR_INVALID_ARGUMENT)])
def test_norm_fp8_refuses(kw, code, fused):
    assert _norm(fused=fused, **kw) == code
    assert tla.last_error()


def test_norm_fp8_residual_and_no_rows():
    assert _norm(res=None) == tla.ERR_INVALID_ARGUMENT
    assert _norm(res=ODD) == tla.ERR_INVALID_ARGUMENT
    assert _norm(T=0, out=None, scales=None, x=None, w=None, res=None) == tla.OK
    assert _norm(T=0, fused=False, out=None, scales=None, x=None, w=None) == tla.OK


def test_norm_fp8_binding_refuses_wrong_tensors():
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(256, dtype=torch.bfloat16)
    out, s = torch.zeros(4, 256, dtype=torch.uint8), torch.zeros(4)
    bad = [
        dict(out=out[:, ::2]), dict(out=out[:3]), dict(s=torch.zeros(3)), dict(s=torch.zeros(4, dtype=torch.float16)),
        dict(s=torch.zeros(4), group=64), dict(x=x[:, ::2]), dict(w=w[:10]), dict(w=w.float()),
        dict(x=x.t().contiguous().t()), dict(res=x.float()), dict(res=x[:2]), dict()]   # the last: not on a GPU
    for kw in bad:
        a = {**dict(x=x, w=w, out=out, s=s, group=0, res=x.clone()), **kw}
        with pytest.raises(tla.TLError):
            tla.fused_add_rms_norm_fp8(a["out"], a["s"], a["res"], a["x"], a["w"], 1e-5, a["group"])
        if "res" not in kw:
            with pytest.raises(tla.TLError):
                tla.rms_norm_fp8(a["out"], a["s"], a["x"], a["w"], 1e-5, a["group"])
