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


def _axes_desc(**kw):
    d = tla.RopeAxesDesc()
    d.num_heads, d.num_kv_heads, d.head_size, d.block_size, d.num_blocks = 8, 2, 128, 16, 64
    d.dtype = d.kv_dtype = tla.BF16
    d.style, d.num_axes, d.interleaved, d.max_positions = tla.ROPE_HALVES, 3, 0, 4096
    d.axis_pairs[0], d.axis_pairs[1], d.axis_pairs[2] = 16, 24, 24
    for k, v in kw.items():
        if k == "axis_pairs":
            for i in range(4):
                d.axis_pairs[i] = v[i] if i < len(v) else 0
        else:
            setattr(d, k, v)
    return d


def _axes(d, T=4, q=FAKE, q_out=FAKE, key=FAKE, value=FAKE, k=FAKE, v=FAKE, ks=None, vs=None, slots=FAKE, pos=FAKE,
          cos=FAKE, sin=FAKE, strides=(0, 0, 0, 0)):
    return L.tl_rope_axes_reshape_and_cache(None if d is None else ctypes.byref(d), q, q_out, key, value, k, v, ks, vs,
                                            slots, pos, cos, sin, T, *strides, None)


@pytest.mark.parametrize("kw,code", [
    (dict(num_kv_heads=0), tla.ERR_INVALID_ARGUMENT), (dict(num_heads=-1), tla.ERR_INVALID_ARGUMENT),
    (dict(head_size=120), tla.ERR_INVALID_ARGUMENT), (dict(head_size=272, axis_pairs=[136]), tla.ERR_NOT_IMPLEMENTED),
    (dict(block_size=0), tla.ERR_INVALID_ARGUMENT), (dict(num_blocks=0), tla.ERR_INVALID_ARGUMENT),
    (dict(max_positions=0), tla.ERR_INVALID_ARGUMENT), (dict(dtype=9), tla.ERR_INVALID_ARGUMENT),
    (dict(dtype=tla.FP8_E4M3, kv_dtype=tla.FP8_E4M3), tla.ERR_INVALID_ARGUMENT),
    (dict(kv_dtype=tla.F16), tla.ERR_NOT_IMPLEMENTED),
    (dict(dtype=tla.F32, kv_dtype=tla.FP8_E4M3), tla.ERR_NOT_IMPLEMENTED),
    (dict(style=2), tla.ERR_INVALID_ARGUMENT), (dict(interleaved=2), tla.ERR_INVALID_ARGUMENT),
    (dict(num_axes=0), tla.ERR_INVALID_ARGUMENT), (dict(num_axes=5), tla.ERR_INVALID_ARGUMENT),
    (dict(axis_pairs=[16, 24, 23]), tla.ERR_INVALID_ARGUMENT), (dict(axis_pairs=[16, 25, 24]), tla.ERR_INVALID_ARGUMENT),
    (dict(axis_pairs=[-1, 41, 24]), tla.ERR_INVALID_ARGUMENT),
    (dict(axis_pairs=[16, 24, 0, 24]), tla.ERR_INVALID_ARGUMENT),      # the fourth is not one of num_axes
    (dict(axis_pairs=[2**31 - 1, 2**31 - 1, 66]), tla.ERR_INVALID_ARGUMENT),
    (dict(num_blocks=2**27, block_size=32), tla.ERR_INVALID_ARGUMENT)])
def test_rope_axes_refuses_descriptors(kw, code):
    assert _axes(_axes_desc(**kw)) == code
    assert tla.last_error()


def test_rope_axes_refuses_arguments():
    assert _axes(None) == tla.ERR_INVALID_ARGUMENT
    d, f = _axes_desc(), _axes_desc(kv_dtype=tla.FP8_E4M3)
    assert _axes(d, T=-1) == tla.ERR_INVALID_ARGUMENT
    for name in ("q", "q_out", "key", "value", "k", "v", "slots", "pos", "cos", "sin"):
        assert _axes(d, **{name: None}) == tla.ERR_INVALID_ARGUMENT, name
    for name in ("q", "q_out", "key", "value", "k", "v"):
        assert _axes(d, **{name: ODD}) == tla.ERR_INVALID_ARGUMENT, name
    assert _axes(d, ks=FAKE, vs=FAKE) == tla.ERR_INVALID_ARGUMENT
    assert _axes(f) == tla.ERR_INVALID_ARGUMENT                        # no scales
    assert _axes(f, ks=FAKE) == tla.ERR_INVALID_ARGUMENT
    assert _axes(f, ks=FAKE, vs=ctypes.c_void_p(0x1002)) == tla.ERR_INVALID_ARGUMENT
    assert _axes(_axes_desc(kv_dtype=tla.FP8_E4M3, head_size=64, axis_pairs=[8, 12, 12]), ks=FAKE, vs=FAKE) \
        == tla.ERR_NOT_IMPLEMENTED
    for i, row in enumerate((8 * 128, 8 * 128, 2 * 128, 2 * 128)):
        s = [0, 0, 0, 0]
        s[i] = row - 1
        assert _axes(d, strides=s) == tla.ERR_INVALID_ARGUMENT
        s[i] = -row
        assert _axes(d, strides=s) == tla.ERR_INVALID_ARGUMENT
    assert _axes(d, T=0, q=None, q_out=None, key=None, value=None, k=None, v=None, slots=None, pos=None, cos=None,
                 sin=None) == tla.OK


def test_fp8_scaled_append_refuses():
    def call(T=4, n_kv=2, D=128, BS=16, N=64, dtype=tla.F16, key=FAKE, value=FAKE, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE,
             slots=FAKE):
        return L.tl_reshape_and_cache_fp8_scaled(key, value, dtype, k, v, ks, vs, slots, T, n_kv, D, BS, N, None)
    for kw in (dict(T=-1), dict(n_kv=0), dict(D=0), dict(BS=0), dict(N=0), dict(key=None), dict(value=None), dict(k=None),
               dict(v=None), dict(ks=None), dict(vs=None), dict(slots=None), dict(key=ODD), dict(value=ODD),
               dict(ks=ctypes.c_void_p(0x1002)), dict(N=2**28, BS=16)):
        assert call(**kw) == tla.ERR_INVALID_ARGUMENT, kw
    for kw in (dict(dtype=tla.F32), dict(dtype=tla.FP8_E4M3), dict(D=64), dict(D=256)):
        assert call(**kw) == tla.ERR_NOT_IMPLEMENTED, kw
    assert call(T=0, key=None, value=None, k=None, v=None, ks=None, vs=None, slots=None) == tla.OK


def test_append_bindings_refuse_wrong_tensors():
    bf, i32, u8 = torch.bfloat16, torch.int32, torch.uint8
    good = dict(q=torch.zeros(4, 8, 128, dtype=bf), key=torch.zeros(4, 2, 128, dtype=bf),
                value=torch.zeros(4, 2, 128, dtype=bf), k=torch.zeros(6, 2, 128, 16, dtype=u8),
                v=torch.zeros(6, 2, 128, 16, dtype=u8), slots=torch.zeros(4, dtype=i32),
                pos=torch.zeros(3, 4, dtype=i32), cos=torch.zeros(99, 64), sin=torch.zeros(99, 64),
                q_out=torch.zeros(4, 8, 128, dtype=bf), ks=torch.zeros(6, 2, 16), vs=torch.zeros(6, 2, 16))
    desc = tla.make_rope_axes_desc(good["q"], good["key"], good["k"], [16, 24, 24], 99)

    def call(**kw):
        a = {**good, **kw}
        tla.rope_axes_reshape_and_cache(desc, a["q"], a["key"], a["value"], a["k"], a["v"], a["slots"], a["pos"],
                                        a["cos"], a["sin"], q_out=a["q_out"], k_scales=a["ks"], v_scales=a["vs"])
    for kw in (dict(q=good["q"][:3]), dict(q=good["q"].half()), dict(q_out=good["q"][:, :4]), dict(key=good["key"][:3]),
               dict(key=good["key"].float()), dict(value=good["value"][:3]), dict(value=good["value"].half()),
               dict(key=torch.zeros(4, 128, 2, dtype=bf).transpose(1, 2)), dict(q=good["q"][:1].expand(4, 8, 128)),
               dict(k=good["k"][:5]), dict(v=good["v"].to(bf)), dict(k=good["k"].transpose(0, 1)),
               dict(slots=good["slots"].long()), dict(slots=good["slots"][:3]), dict(pos=good["pos"][:2]),
               dict(pos=torch.zeros(4, 3, dtype=i32).t()), dict(cos=good["cos"][:98]), dict(sin=good["sin"].double()),
               dict(ks=good["ks"][:5]), dict(vs=good["vs"].half()), dict()):      # the last: not on a GPU
        with pytest.raises(tla.TLError):
            call(**kw)
    for bad in ([], [1] * 5):
        with pytest.raises(tla.TLError):
            tla.make_rope_axes_desc(good["q"], good["key"], good["k"], bad, 99)
    for kw in (dict(key=good["key"][:3]), dict(value=good["value"].half()), dict(ks=good["ks"].half()),
               dict(k=good["k"].to(bf), v=good["v"].to(bf)), dict(slots=good["slots"].long()), dict()):
        a = {**good, **kw}
        with pytest.raises(tla.TLError):
            tla.reshape_and_cache_fp8_scaled(a["key"], a["value"], a["k"], a["v"], a["ks"], a["vs"], a["slots"])


def _decode_desc(**kw):
    d = tla.DecodeDesc()
    d.num_seqs, d.num_heads, d.num_kv_heads, d.head_size, d.block_size = 4, 32, 8, 128, 16
    d.max_blocks_per_seq, d.num_blocks, d.q_dtype, d.kv_dtype = 64, 512, tla.BF16, tla.FP8_E4M3
    d.gqa_map, d.partition_tokens, d.scale = tla.GQA_GROUPED, 0, 0.088
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _decode(d, out=FAKE, q=FAKE, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, bt=FAKE, sl=FAKE, ctx=1024, ws=None, ws_bytes=0):
    return L.tl_paged_attention_decode_scaled(None if d is None else ctypes.byref(d), out, q, k, v, ks, vs, bt, sl, ctx, ws,
                                              ws_bytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(kv_dtype=tla.BF16), tla.ERR_INVALID_ARGUMENT), (dict(kv_dtype=0, q_dtype=0), tla.ERR_INVALID_ARGUMENT),
    (dict(q_dtype=tla.F32), tla.ERR_NOT_IMPLEMENTED), (dict(head_size=64), tla.ERR_NOT_IMPLEMENTED),
    (dict(head_size=256), tla.ERR_NOT_IMPLEMENTED), (dict(block_size=12), tla.ERR_NOT_IMPLEMENTED),
    (dict(block_size=512), tla.ERR_NOT_IMPLEMENTED), (dict(num_heads=30), tla.ERR_INVALID_ARGUMENT),
    (dict(num_kv_heads=0), tla.ERR_INVALID_ARGUMENT), (dict(num_blocks=0), tla.ERR_INVALID_ARGUMENT),
    (dict(gqa_map=2), tla.ERR_INVALID_ARGUMENT), (dict(partition_tokens=100), tla.ERR_INVALID_ARGUMENT),
    (dict(num_seqs=-1), tla.ERR_INVALID_ARGUMENT)])
def test_scaled_decode_refuses_descriptors(kw, code):
    assert _decode(_decode_desc(**kw)) == code
    assert tla.last_error()


def test_scaled_decode_refuses_arguments():
    d = _decode_desc()
    assert _decode(None) == tla.ERR_INVALID_ARGUMENT
    for name in ("out", "q", "k", "v", "ks", "vs", "bt", "sl"):
        assert _decode(d, **{name: None}) == tla.ERR_INVALID_ARGUMENT, name
    for name in ("k", "v", "ks", "vs"):
        assert _decode(d, **{name: ctypes.c_void_p(0x1002)}) == tla.ERR_INVALID_ARGUMENT, name
    assert _decode(d, ctx=-1) == tla.ERR_INVALID_ARGUMENT
    assert _decode(_decode_desc(partition_tokens=256)) == tla.ERR_INVALID_ARGUMENT      # no workspace
    assert _decode(_decode_desc(partition_tokens=256), ws=FAKE, ws_bytes=64) == tla.ERR_INVALID_ARGUMENT
    assert _decode(_decode_desc(num_seqs=0), out=None, q=None, k=None, v=None, ks=None, vs=None, bt=None, sl=None) == tla.OK


def test_scaled_decode_binding_refuses_wrong_tensors():
    bf, i32, u8 = torch.bfloat16, torch.int32, torch.uint8
    good = dict(q=torch.zeros(3, 8, 128, dtype=bf), out=torch.zeros(3, 8, 128, dtype=bf),
                k=torch.zeros(6, 2, 128, 16, dtype=u8), v=torch.zeros(6, 2, 128, 16, dtype=u8), ks=torch.zeros(6, 2, 16),
                vs=torch.zeros(6, 2, 16), bt=torch.zeros(3, 5, dtype=i32), sl=torch.zeros(3, dtype=i32))
    desc = tla.make_decode_desc(good["q"], good["k"], good["bt"], 2, 0.1)
    for kw in (dict(q=good["q"][:2]), dict(q=good["q"].half()), dict(out=good["out"].float()),
               dict(out=good["out"].transpose(0, 1)), dict(k=good["k"][:5]), dict(v=good["v"].view(6, 2, 16, 128)),
               dict(ks=good["ks"][:, :1]), dict(vs=good["vs"].half()), dict(bt=good["bt"].long()),
               dict(bt=good["bt"][:, :4]), dict(sl=good["sl"][:2]), dict()):            # the last: not on a GPU
        a = {**good, **kw}
        with pytest.raises(tla.TLError):
            tla.paged_attention_decode_scaled(desc, a["out"], a["q"], a["k"], a["v"], a["ks"], a["vs"], a["bt"], a["sl"],
                                              80)


def _prefill_desc(**kw):
    d = tla.PrefillDesc()
    d.num_seqs, d.num_heads, d.num_kv_heads, d.head_size, d.block_size = 4, 32, 8, 128, 16
    d.max_blocks_per_seq, d.num_blocks, d.dtype, d.kv_dtype = 64, 512, tla.BF16, tla.FP8_E4M3
    d.gqa_map, d.scale = tla.GQA_GROUPED, 0.088
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _prefill(d, out=FAKE, q=FAKE, cu=FAKE, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, bt=FAKE, sl=FAKE, total=64, most=32):
    return L.tl_chunked_prefill_scaled(None if d is None else ctypes.byref(d), out, q, cu, k, v, ks, vs, bt, sl, total, most,
                                       None)


@pytest.mark.parametrize("kw,code", [
    (dict(kv_dtype=tla.BF16), tla.ERR_INVALID_ARGUMENT), (dict(kv_dtype=0), tla.ERR_INVALID_ARGUMENT),
    (dict(dtype=tla.F32), tla.ERR_NOT_IMPLEMENTED), (dict(head_size=64), tla.ERR_NOT_IMPLEMENTED),
    (dict(block_size=4), tla.ERR_NOT_IMPLEMENTED), (dict(block_size=24), tla.ERR_NOT_IMPLEMENTED),
    (dict(num_heads=30), tla.ERR_INVALID_ARGUMENT), (dict(num_blocks=0), tla.ERR_INVALID_ARGUMENT),
    (dict(num_prefill_seqs=5), tla.ERR_INVALID_ARGUMENT), (dict(scale=0.0), tla.ERR_INVALID_ARGUMENT),
    (dict(scale=float("nan")), tla.ERR_INVALID_ARGUMENT), (dict(gqa_map=3), tla.ERR_INVALID_ARGUMENT)])
def test_scaled_prefill_refuses_descriptors(kw, code):
    assert _prefill(_prefill_desc(**kw)) == code
    assert tla.last_error()


def test_scaled_prefill_refuses_arguments():
    d = _prefill_desc()
    assert _prefill(None) == tla.ERR_INVALID_ARGUMENT
    for name in ("out", "q", "cu", "k", "v", "ks", "vs", "bt", "sl"):
        assert _prefill(d, **{name: None}) == tla.ERR_INVALID_ARGUMENT, name
    for name in ("q", "k", "v", "ks", "vs", "out"):
        assert _prefill(d, **{name: ctypes.c_void_p(0x1002)}) == tla.ERR_INVALID_ARGUMENT, name
    assert _prefill(d, total=16, most=17) == tla.ERR_INVALID_ARGUMENT
    assert _prefill(d, total=-1) == tla.ERR_INVALID_ARGUMENT
    assert _prefill(d, total=0, most=0, out=None, q=None, ks=None, vs=None) == tla.OK


def test_scaled_prefill_binding_refuses_wrong_tensors():
    bf, i32, u8 = torch.bfloat16, torch.int32, torch.uint8
    good = dict(q=torch.zeros(9, 8, 128, dtype=bf), out=torch.zeros(9, 8, 128, dtype=bf), cu=torch.zeros(4, dtype=i32),
                k=torch.zeros(6, 2, 128, 16, dtype=u8), v=torch.zeros(6, 2, 128, 16, dtype=u8), ks=torch.zeros(6, 2, 16),
                vs=torch.zeros(6, 2, 16), bt=torch.zeros(3, 5, dtype=i32), sl=torch.zeros(3, dtype=i32))
    desc = tla.make_prefill_desc(good["q"], good["k"], good["bt"], 3, 2, 0.1, kv_dtype=tla.FP8_E4M3)
    for kw in (dict(q=good["q"].half()), dict(out=good["out"][:8]), dict(q=good["q"][:, :4], out=good["out"][:, :4]),
               dict(cu=good["cu"][:3]), dict(cu=good["cu"].long()), dict(k=good["k"][:5]), dict(ks=good["ks"].half()),
               dict(vs=good["vs"][:, :, :8]), dict(bt=good["bt"][:2]), dict(sl=good["sl"].long()), dict()):
        a = {**good, **kw}
        with pytest.raises(tla.TLError):
            tla.chunked_prefill_scaled(desc, a["out"], a["q"], a["cu"], a["k"], a["v"], a["ks"], a["vs"], a["bt"], a["sl"], 4)


def test_appends_refuse_rows_and_strides_past_int32():
    d = _axes_desc(num_heads=2**24)
    assert _axes(d) == tla.ERR_INVALID_ARGUMENT
    assert _axes(_axes_desc(num_kv_heads=2**24)) == tla.ERR_INVALID_ARGUMENT
    assert L.tl_reshape_and_cache_fp8_scaled(FAKE, FAKE, tla.F16, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 2**24, 128, 16, 64,
                                             None) == tla.ERR_INVALID_ARGUMENT
    far = torch.empty(2**31 + 256, dtype=torch.bfloat16, device="meta").as_strided((2, 2, 128), (2**31, 128, 1))
    with pytest.raises(tla.TLError, match="tokens less than 2\\^31 apart"):
        tla._token_stride(far, 2, 2, 128, tla.BF16, "key")
    assert tla._token_stride(far[:, :, :].as_strided((2, 2, 128), (2**31 - 1, 128, 1)), 2, 2, 128, tla.BF16, "key") \
        == 2**31 - 1


def test_rope_axes_refuses_two_strides_in_place():
    # one token has none; the others would be read where an earlier one was written
    d = _axes_desc()
    assert _axes(d, strides=(2048, 1024, 0, 0)) == tla.ERR_INVALID_ARGUMENT
    assert _axes(d, strides=(0, 2048, 0, 0)) == tla.ERR_INVALID_ARGUMENT


def test_scaled_decode_refuses_a_strided_workspace():
    bf, i32, u8 = torch.bfloat16, torch.int32, torch.uint8
    q, pool, scales = torch.zeros(3, 8, 128, dtype=bf), torch.zeros(6, 2, 128, 16, dtype=u8), torch.zeros(6, 2, 16)
    tables, lens = torch.zeros(3, 5, dtype=i32), torch.zeros(3, dtype=i32)
    desc = tla.make_decode_desc(q, pool, tables, 2, 0.1)
    with pytest.raises(tla.TLError, match="workspace"):
        tla.paged_attention_decode_scaled(desc, q.clone(), q, pool, pool, scales, scales, tables, lens, 80,
                                          torch.zeros(1, dtype=u8).expand(1 << 20))
