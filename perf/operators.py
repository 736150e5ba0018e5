"""The operators of an 8-bit serving step: what is measured of them, and their plain forms.

A layer of a decoder whose cache is FP8 with a scale for each token and head,
found as the token is written: the norm that hands an FP8 product its operand,
rotary positions with one or several axes on the way into the pools, the
quantising append, and the attention that reads the scaled pools back, for
single tokens and for chunks of a prompt.

Where `own` is false, run() computes them in elementary torch operations in 32
bits, rounded once; where it is true, it calls tl_attn.  Codes come back as
float8 tensors, next to the scales that they are held under.
"""
import functools
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
FP8_MAX = 448.0
EPS = 1e-5
ROPE_BASE = 10000.0
ADJACENT, HALVES = 0, 1


@functools.cache
def lib():
    """The framework's binding, imported once."""
    sys.path.insert(0, os.path.join(os.getcwd(), "truellm-engine_amd"))
    import tl_attn
    return tl_attn


def listed():
    return [
        # The norm before a layer's products in a decode step: 64 sequences,
        # residual added, one scale for each token.
        dict(name="norm_step", kind="norm", rows=64, hidden=4096, dtype="bf16", fused=True, group=0),
        # A prompt chunk through a wide model, a scale for each 128 channels.
        dict(name="norm_prompt", kind="norm", rows=4096, hidden=8192, dtype="bf16", fused=True, group=128),
        # The first norm of a model (nothing to add yet), odd sizes.
        dict(name="norm_first", kind="norm", rows=333, hidden=5632, dtype="f16", fused=False, group=0),
        # A decode step of a model with time, height and width axes, dealt in
        # turn over the pairs.
        dict(name="axes_step", kind="append", seqs=64, tokens=1, heads=32, kv_heads=8, head=128, block=16,
             dtype="f16", kv="same", axes="24,20,20", interleaved=True, style=HALVES),
        # Prompts with images in them: runs of text and grids of patches.
        dict(name="axes_prompt", kind="append", seqs=6, tokens=700, heads=32, kv_heads=8, head=128, block=16,
             dtype="bf16", kv="same", axes="16,24,24", interleaved=False, style=HALVES),
        # The step's keys and values into FP8 pools, scales found on the way.
        dict(name="quant_step", kind="append", seqs=64, tokens=1, heads=32, kv_heads=8, head=128, block=16,
             dtype="f16", kv="fp8", axes="64", interleaved=False, style=ADJACENT),
        # The same for prompts, image tokens among them, in larger blocks.
        dict(name="quant_prompt", kind="append", seqs=5, tokens=811, heads=64, kv_heads=8, head=128, block=32,
             dtype="bf16", kv="fp8", axes="16,24,24", interleaved=False, style=HALVES),
        # One user's next token.
        dict(name="decode_one", kind="decode", batch=1, ctx=4096, heads=32, kv_heads=8, block=16, dtype="f16",
             ragged=False),
        # A full batch at one length.
        dict(name="decode_batch", kind="decode", batch=64, ctx=4096, heads=32, kv_heads=8, block=16, dtype="bf16",
             ragged=False),
        # Few sequences of every length up to a long context, the 64-head shape.
        dict(name="decode_long", kind="decode", batch=16, ctx=32768, heads=64, kv_heads=8, block=32, dtype="f16",
             ragged=True),
        # One user's prompt after an earlier part of it: time to first token.
        dict(name="chunk_one_user", kind="chunk", prompts=1, chunk=500, ctx=1500, decodes=0, heads=32, kv_heads=8,
             block=16, dtype="f16"),
        # A scheduler's mixed batch: the last chunk of eight prompts, and
        # decode rows beside them.
        dict(name="chunk_mixed", kind="chunk", prompts=8, chunk=512, ctx=2048, decodes=32, heads=64, kv_heads=8,
             block=16, dtype="bf16"),
    ]


def log_int(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "append", "append", "decode", "decode", "chunk"])
    dtype = rng.choice(["f16", "bf16"])
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (32, 32), (16, 2), (8, 1), (12, 4)])
    block = rng.choice([8, 16, 16, 32, 64, 128, 256])
    if kind == "norm":
        hidden = rng.choice([4096, 8192, 2048, 5632, 14336, 8 * log_int(rng, 8, 1024)])
        group = rng.choice([0, 0, 32, 64, 128, 256])
        return dict(kind=kind, rows=log_int(rng, 1, 4096 * 8192 // max(hidden, 8192)), hidden=hidden,
                    dtype=rng.choice([dtype, dtype, "f32"]), fused=rng.random() < 0.6,
                    group=group if group and hidden % group == 0 else 0)
    if kind == "append":
        seqs = log_int(rng, 1, 64)
        tokens = 1 if rng.random() < 0.4 else log_int(rng, 1, 4200 // seqs)
        kv = rng.choice(["same", "fp8", "fp8"])
        head = 128 if kv == "fp8" or rng.random() < 0.7 else 64
        axes, dealt = rng.choice([("64", False), ("16,24,24", False), ("24,20,20", True), ("21,21,22", False),
                                  ("32,32", True)] if head == 128 else
                                 [("32", False), ("8,12,12", False), ("12,10,10", True)])
        return dict(kind=kind, seqs=seqs, tokens=tokens, heads=heads, kv_heads=kv_heads, head=head, block=block,
                    dtype=dtype, kv=kv, axes=axes, interleaved=dealt, style=rng.choice([ADJACENT, HALVES]))
    if kind == "decode":
        batch = log_int(rng, 1, 64)
        most = min(32768, 64 * 4096 * 8 // (batch * kv_heads))
        return dict(kind=kind, batch=batch, ctx=log_int(rng, 1, most), heads=heads, kv_heads=kv_heads, block=block,
                    dtype=dtype, ragged=rng.random() < 0.6)
    prompts = log_int(rng, 1, 8)
    chunk = log_int(rng, 2, 4096 // prompts)
    ctx = chunk if rng.random() < 0.4 else min(chunk + log_int(rng, 1, 6000), 8192 * 2048 // (prompts * chunk))
    return dict(kind=kind, prompts=prompts, chunk=chunk, ctx=max(ctx, chunk), decodes=rng.choice([0, 0, 3, 17]),
                heads=heads, kv_heads=kv_heads, block=block, dtype=dtype)


# ---------------------------------------------------------------------------
# what the cases are made of
# ---------------------------------------------------------------------------

def case_rng(case):
    return random.Random("|".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"))


def lengths(case):
    """Sequence lengths of a decode batch: all of ctx, or spread below it, a sequence without tokens among many."""
    n, ctx = case["batch"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * n
    rng = case_rng(case)
    lens = [ctx] + [rng.randint(max(1, ctx // 16), ctx) for _ in range(n - 1)]
    if n >= 20:
        lens[n // 2] = 0
    return lens


def chunk_rows(case):
    """(new tokens, context) of each prompt, then of each decode row."""
    rng = case_rng(case)
    rows = []
    for i in range(case["prompts"]):
        cut = 0 if i == 0 or case["prompts"] == 8 else rng.randint(0, case["chunk"] // 2)
        rows.append((max(2, case["chunk"] - cut), max(2, case["ctx"] - cut)))
    return rows + [(1, max(1, case["ctx"] - i)) for i in range(case["decodes"])]


def append_spans(case):
    """(first position, tokens) of each sequence of an append: it begins anywhere in a block."""
    rng = case_rng(case)
    return [(rng.randint(0, 3 * case["block"]),
             case["tokens"] if case["tokens"] < 16 or i == 0 else case["tokens"] - rng.randint(0, 7))
            for i in range(case["seqs"])]


def axes_of(case):
    return [int(n) for n in case["axes"].split(",")]


def axis_of_pair(case):
    """The axis that turns each pair: runs of consecutive pairs, or the axes in turn while they have pairs left."""
    left = axes_of(case)
    if not case["interleaved"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    got = []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                got.append(a)
    return got


def axis_positions(case):
    """positions[axis][token]: text advances on every axis; a grid of patches in each longer sequence has its row and
    column on the later axes."""
    n_axes, rows = len(axes_of(case)), []
    for at, n in append_spans(case):
        grid = range(n // 4, n // 4 + n // 2) if n >= 8 and n_axes > 1 else range(0)
        wide = max(1, math.isqrt(len(grid)))
        row, shift = [], 0
        for i in range(n):
            if i in grid:
                k = i - grid.start
                place = [at + grid.start] + [at + grid.start + d for d in (k // wide, k % wide, k % 2)]
                shift = len(grid) - wide if k == len(grid) - 1 else 0
            else:
                place = [at + i - shift] * 4
            row.append(place[:n_axes])
        rows += row
    return [list(axis) for axis in zip(*rows)]


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, g):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g)


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def tables_for(blocks, total, g):
    """Block tables over a pool of `total` blocks in a free list's order: row s holds blocks[s] ids, then -1."""
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    t = torch.full((len(blocks), max(1, max(blocks))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(blocks):
        t[s, :n] = order[at:at + n]
        at += n
    return t


def block_counts(lens, bs):
    return [(n + bs - 1) // bs for n in lens]


def pool_blocks(blocks):
    return math.ceil(1.25 * sum(blocks)) + 1


def scaled_pool(n_blocks, kv_heads, head, bs, g):
    """Codes [n, kv_heads, head, bs] and scales [n, kv_heads, bs] of rows N(0, 1) times a size of their own."""
    codes = torch.empty((n_blocks, kv_heads, head, bs), dtype=torch.uint8, device="cuda")
    scales = torch.empty((n_blocks, kv_heads, bs), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // (kv_heads * head * bs))
    for i in range(0, n_blocks, step):
        x = normal(codes[i:i + step].shape, torch.float32, g)
        x *= normal(scales[i:i + step].shape, torch.float32, g).mul_(0.4).exp_().unsqueeze(2)
        scales[i:i + step] = x.abs().amax(2) / FP8_MAX
        x /= scales[i:i + step].unsqueeze(2)
        codes[i:i + step] = x.clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, scales


def rope_tables(n, head):
    inv = ROPE_BASE ** (-torch.arange(0, head, 2, device="cuda", dtype=torch.float64) / head)
    a = torch.outer(torch.arange(n, device="cuda", dtype=torch.float64), inv)
    return a.cos().float().contiguous(), a.sin().float().contiguous()


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------

def prepare(case, seed):
    s = {"norm": prepare_norm, "append": prepare_append, "decode": prepare_decode,
         "chunk": prepare_chunk}[case["kind"]](case, generator(seed))
    s["case"] = case
    return s


def prepare_norm(case, g):
    rows, hidden, dtype = case["rows"], case["hidden"], DTYPES[case["dtype"]]
    groups = hidden // case["group"] if case["group"] else 1
    return dict(x=normal((rows, hidden), dtype, g), residual=normal((rows, hidden), dtype, g),
                weight=(1.0 + 0.1 * normal((hidden,), torch.float32, g)).to(dtype),
                out=torch.empty((rows, hidden), dtype=torch.uint8, device="cuda"),
                scales=torch.empty((rows, groups) if case["group"] else (rows,), dtype=torch.float32, device="cuda"))


def prepare_append(case, g):
    spans, bs, H, n_kv, D = append_spans(case), case["block"], case["heads"], case["kv_heads"], case["head"]
    dtype = DTYPES[case["dtype"]]
    blocks = block_counts([a + n for a, n in spans], bs)
    total = pool_blocks(blocks)
    tables = tables_for(blocks, total, g)
    T = sum(n for _, n in spans)
    at = torch.cat([torch.arange(a, a + n, device="cuda") for a, n in spans])
    seq = torch.cat([torch.full((n,), i, device="cuda") for i, (_, n) in enumerate(spans)])
    slots = (tables[seq, at // bs].long() * bs + at % bs).to(torch.int32)
    positions = int32(axis_positions(case))
    cos, sin = rope_tables(max(a + n for a, n in spans), D)
    s = dict(q=normal((T, H, D), dtype, g), key=normal((T, n_kv, D), dtype, g), value=normal((T, n_kv, D), dtype, g),
             slots=slots, positions=positions, cos=cos, sin=sin, k_scales=None, v_scales=None)
    s["q_out"] = torch.empty_like(s["q"])
    # a few key channels are larger than the rest
    loud = torch.ones((n_kv, D), dtype=dtype, device="cuda")
    loud[:, ::31] = 6.0
    s["key"] *= loud
    if case["kv"] == "fp8":
        s["k"], s["k_scales"] = scaled_pool(total, n_kv, D, bs, g)
        s["v"], s["v_scales"] = scaled_pool(total, n_kv, D, bs, g)
    else:
        s["k"], s["v"] = normal((total, n_kv, D, bs), dtype, g), normal((total, n_kv, D, bs), dtype, g)
    s["axis"] = torch.tensor(axis_of_pair(case), device="cuda")
    if own:
        s["desc"] = lib().make_rope_axes_desc(s["q"], s["key"], s["k"], axes_of(case), cos.shape[0],
                                              style=case["style"], interleaved=case["interleaved"])
    return s


def prepare_decode(case, g):
    lens, bs, H, n_kv = lengths(case), case["block"], case["heads"], case["kv_heads"]
    blocks = block_counts(lens, bs)
    total = pool_blocks(blocks)
    s = dict(tables=tables_for(blocks, total, g), lens=int32(lens), max_ctx=max(lens),
             q=normal((case["batch"], H, 128), DTYPES[case["dtype"]], g))
    s["k"], s["k_scales"] = scaled_pool(total, n_kv, 128, bs, g)
    s["v"], s["v_scales"] = scaled_pool(total, n_kv, 128, bs, g)
    s["out"] = torch.empty_like(s["q"])
    if own:
        tla = lib()
        s["desc"] = tla.make_decode_desc(s["q"], s["k"], s["tables"], n_kv, 1.0 / math.sqrt(128))
        s["ws"] = torch.empty(max(16, tla.workspace_bytes(s["desc"], s["max_ctx"])), dtype=torch.uint8,
                              device="cuda")
    return s


def prepare_chunk(case, g):
    rows, bs, H, n_kv = chunk_rows(case), case["block"], case["heads"], case["kv_heads"]
    blocks = block_counts([c for _, c in rows], bs)
    total = pool_blocks(blocks)
    starts = [0]
    for n, _ in rows:
        starts.append(starts[-1] + n)
    s = dict(tables=tables_for(blocks, total, g), lens=int32([c for _, c in rows]), cu=int32(starts),
             max_q=max(n for n, _ in rows), max_ctx=max(c for _, c in rows),
             q=normal((starts[-1], H, 128), DTYPES[case["dtype"]], g))
    s["k"], s["k_scales"] = scaled_pool(total, n_kv, 128, bs, g)
    s["v"], s["v_scales"] = scaled_pool(total, n_kv, 128, bs, g)
    s["out"] = torch.empty_like(s["q"])
    if own:
        s["desc"] = lib().make_prefill_desc(s["q"], s["k"], s["tables"], len(rows), n_kv, 1.0 / math.sqrt(128),
                                            num_prefill_seqs=case["prompts"], kv_dtype=lib().FP8_E4M3)
    return s


# ---------------------------------------------------------------------------
# run
# ---------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"norm": own_norm, "append": own_append, "decode": own_decode, "chunk": own_chunk}[kind](s, lib())
    return {"norm": plain_norm, "append": plain_append, "decode": plain_decode, "chunk": plain_chunk}[kind](s)


def as_fp8(codes):
    return codes.view(torch.float8_e4m3fn)


def own_norm(s, tla):
    case = s["case"]
    if case["fused"]:
        tla.fused_add_rms_norm_fp8(s["out"], s["scales"], s["residual"], s["x"], s["weight"], EPS, case["group"])
    else:
        tla.rms_norm_fp8(s["out"], s["scales"], s["x"], s["weight"], EPS, case["group"])
    return [as_fp8(s["out"]), s["scales"], s["residual"]]


def own_append(s, tla):
    tla.rope_axes_reshape_and_cache(s["desc"], s["q"], s["key"], s["value"], s["k"], s["v"], s["slots"],
                                    s["positions"], s["cos"], s["sin"], q_out=s["q_out"], k_scales=s["k_scales"],
                                    v_scales=s["v_scales"])
    return appended(s)


def appended(s):
    if s["case"]["kv"] == "fp8":
        return [s["q_out"], as_fp8(s["k"]), as_fp8(s["v"]), s["k_scales"], s["v_scales"]]
    return [s["q_out"], s["k"], s["v"]]


def own_decode(s, tla):
    tla.paged_attention_decode_scaled(s["desc"], s["out"], s["q"], s["k"], s["v"], s["k_scales"], s["v_scales"],
                                      s["tables"], s["lens"], s["max_ctx"], s["ws"])
    return [s["out"]]


def own_chunk(s, tla):
    tla.chunked_prefill_scaled(s["desc"], s["out"], s["q"], s["cu"], s["k"], s["v"], s["k_scales"], s["v_scales"],
                               s["tables"], s["lens"], s["max_q"])
    return [s["out"]]


# ---- plain forms --------------------------------------------------------------

def plain_norm(s):
    case, x, rows = s["case"], s["x"].float(), s["case"]["rows"]
    if case["fused"]:
        x = x + s["residual"].float()
        s["residual"].copy_(x)
    mean = x.square().mean(-1, keepdim=True)
    if case["fused"]:
        x = s["residual"].float()
    y = x * torch.rsqrt(mean + EPS) * s["weight"].float()
    g = y.view(rows, -1, case["group"] or case["hidden"])
    scale = g.abs().amax(-1, keepdim=True) / FP8_MAX
    codes = (g / scale).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(rows, -1)
    return [codes, scale.view(s["scales"].shape), s["residual"]]


def turned(x, c, s, style):
    """Rows x [T, heads, D] by c, s [T, 1, D / 2]."""
    if style == ADJACENT:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def plain_append(s):
    case, bs = s["case"], s["case"]["block"]
    pair = torch.arange(case["head"] // 2, device="cuda")
    pos = s["positions"].long()[s["axis"]].t()                         # [T, D / 2]
    c, sn = s["cos"][pos, pair].unsqueeze(1), s["sin"][pos, pair].unsqueeze(1)
    s["q_out"].copy_(turned(s["q"].float(), c, sn, case["style"]))
    rows = (turned(s["key"].float(), c, sn, case["style"]), s["value"].float())
    slots = s["slots"].long()
    blk, off = slots // bs, slots % bs
    if case["kv"] != "fp8":
        s["k"][blk, :, :, off] = rows[0].to(s["k"].dtype)
        s["v"][blk, :, :, off] = rows[1].to(s["v"].dtype)
        return appended(s)
    k_scale, v_scale = rows[0].abs().amax(-1) / FP8_MAX, rows[1].abs().amax(-1) / FP8_MAX
    s["k"][blk, :, :, off] = to_codes(rows[0], k_scale)
    s["v"][blk, :, :, off] = to_codes(rows[1], v_scale)
    s["k_scales"][blk, :, off] = k_scale
    s["v_scales"][blk, :, off] = v_scale
    return appended(s)


def to_codes(x, scale):
    return (x / scale.unsqueeze(-1)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(torch.uint8)


def gathered(codes, scales, tables):
    """[seqs, kv_heads, D, tokens] in 32 bits of the sequences' blocks."""
    t = tables.clamp(min=0).long()
    x = as_fp8(codes)[t].float() * scales[t].unsqueeze(3)              # [S, blocks, kv_heads, D, bs]
    return x.permute(0, 2, 3, 1, 4).flatten(3)


def attend(q, k, v, mask):
    """q [S, n, H, D] in 32 bits over k, v [S, kv_heads, D, L]; mask [S, n, L] true where a key is seen."""
    S, n, H, D = q.shape
    n_kv = k.shape[1]
    group = H // n_kv
    qq = q.view(S, n, n_kv, group, D).permute(0, 2, 1, 3, 4).reshape(S, n_kv, n * group, D)
    sc = torch.matmul(qq, k).view(S, n_kv, n, group, -1) / math.sqrt(D)
    sc = sc.masked_fill(~mask[:, None, :, None, :], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, torch.ones_like(total))).view(S, n_kv, n * group, -1)
    o = torch.matmul(v, p.transpose(2, 3).contiguous())                # [S, n_kv, D, n group]
    return o.view(S, n_kv, D, n, group).permute(0, 3, 1, 4, 2).reshape(S, n, H, D)


def plain_decode(s):
    k, v = gathered(s["k"], s["k_scales"], s["tables"]), gathered(s["v"], s["v_scales"], s["tables"])
    seen = torch.arange(k.shape[3], device="cuda")[None, None, :] < s["lens"][:, None, None]
    s["out"].copy_(attend(s["q"].float().unsqueeze(1), k, v, seen).squeeze(1))
    return [s["out"]]


def plain_chunk(s):
    case = s["case"]
    plain_part(s, 0, case["prompts"], s["max_q"])
    if case["decodes"]:
        plain_part(s, case["prompts"], case["prompts"] + case["decodes"], 1)
    return [s["out"]]


def plain_part(s, first, end, most):
    """Sequences first .. end - 1 as a padded batch of `most` queries each."""
    tables, lens, cu = s["tables"][first:end], s["lens"][first:end, None].long(), s["cu"].long()
    n = (cu[first + 1:end + 1] - cu[first:end])[:, None]
    i = torch.arange(most, device="cuda")[None, :]
    row = (cu[first:end, None] + i).clamp(max=s["q"].shape[0] - 1)
    k, v = gathered(s["k"], s["k_scales"], tables), gathered(s["v"], s["v_scales"], tables)
    seen = torch.arange(k.shape[3], device="cuda")[None, None, :] <= (lens - n + i)[:, :, None]
    out = attend(s["q"][row].float(), k, v, seen)
    there = i < n
    s["out"][row[there]] = out[there].to(s["out"].dtype)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    e = 4 if case["dtype"] == "f32" else 2
    if kind == "norm":
        rows, hidden = case["rows"], case["hidden"]
        groups = hidden // case["group"] if case["group"] else 1
        return {"bytes": rows * hidden * (e * (3 if case["fused"] else 1) + 1) + hidden * e + 4 * rows * groups,
                "flops": rows * hidden * 7}
    if kind == "append":
        T, H, n_kv, D = sum(n for _, n in append_spans(case)), case["heads"], case["kv_heads"], case["head"]
        pool = 2 * n_kv * (D + 4) if case["kv"] == "fp8" else 2 * n_kv * D * e
        places = len(set(zip(*axis_positions(case))))
        return {"bytes": T * (2 * H * D * e + 2 * n_kv * D * e + pool + 4 + 4 * len(axes_of(case))) + places * D * 4,
                "flops": T * D * (3 * (H + n_kv) + 4 * n_kv)}
    H, n_kv = case["heads"], case["kv_heads"]
    rows = [(1, n) for n in lengths(case)] if kind == "decode" else chunk_rows(case)
    keys, queries = sum(c for _, c in rows), sum(n for n, _ in rows)
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in rows)
    blocks = sum(block_counts([c for _, c in rows], case["block"]))
    return {"bytes": keys * n_kv * 2 * (128 + 4) + 2 * queries * H * 128 * e + 4 * (blocks + 2 * len(rows)),
            "flops": 4 * pairs * H * 128}


# ---------------------------------------------------------------------------
# the same from the definition, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        return {"norm": exact_norm, "append": exact_append, "decode": exact_attention,
                "chunk": exact_attention}[case["kind"]](case, prepare(case, seed))


def exact_norm(case, s):
    x, w = s["x"].double(), s["weight"].double()
    kept = s["residual"].double()
    if case["fused"]:
        x = kept = x + kept
    inv = 1.0 / torch.sqrt((x * x).sum(1) / case["hidden"] + EPS)
    if case["fused"]:
        x = x.to(DTYPES[case["dtype"]]).double()                       # the norm is of the residual as stored
    y = x * inv[:, None] * w[None, :]
    parts = y.split(case["group"] or case["hidden"], dim=1)
    scale = torch.stack([p.abs().max(1).values for p in parts], 1) / FP8_MAX
    # what a code stands for before it is rounded
    codes = torch.cat([p / scale[:, i:i + 1] for i, p in enumerate(parts)], 1)
    return [codes, scale if case["group"] else scale[:, 0], kept]


def exact_append(case, s):
    T, D, half, bs = s["q"].shape[0], case["head"], case["head"] // 2, case["block"]
    axis, pos = axis_of_pair(case), s["positions"].long()
    c = torch.stack([s["cos"].double()[pos[axis[i]], i] for i in range(half)], 1)[:, None, :]
    sn = torch.stack([s["sin"].double()[pos[axis[i]], i] for i in range(half)], 1)[:, None, :]
    first = [2 * i if case["style"] == ADJACENT else i for i in range(half)]
    second = [i + 1 if case["style"] == ADJACENT else i + half for i in first]

    def rot(x):
        x = x.double()
        y = torch.empty_like(x)
        y[..., first] = x[..., first] * c - x[..., second] * sn
        y[..., second] = x[..., first] * sn + x[..., second] * c
        return y

    slots = s["slots"].long()
    out = [rot(s["q"])]
    pools, scales = [], []
    for pool, kept, rows in ((s["k"], s["k_scales"], rot(s["key"])), (s["v"], s["v_scales"], s["value"].double())):
        if kept is not None:
            scale = rows.abs().max(2).values / FP8_MAX
            rows = rows / scale[:, :, None]
            kept = kept.double()
            kept[slots // bs, :, slots % bs] = scale
            scales.append(kept)
            pool = as_fp8(pool).float()
        pool = pool.double()
        pool[slots // bs, :, :, slots % bs] = rows
        pools.append(pool)
    return out + pools + scales


def exact_attention(case, s):
    H, n_kv, D, bs = case["heads"], case["kv_heads"], 128, case["block"]
    rows = [(1, n) for n in lengths(case)] if case["kind"] == "decode" else chunk_rows(case)
    group, out, at = H // n_kv, torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for j, (n, length) in enumerate(rows):
        if length:
            ids = s["tables"][j, :(length + bs - 1) // bs].long()
            place = length - n + torch.arange(n, device="cuda")
            for h in range(n_kv):
                k, v = ((as_fp8(pool[ids, h]).double() * sc[ids, h].double()[:, None, :]).transpose(0, 1).flatten(1)
                        [:, :length] for pool, sc in ((s["k"], s["k_scales"]), (s["v"], s["v_scales"])))
                q = s["q"][at:at + n, h * group:(h + 1) * group].double().reshape(n * group, D)
                sc = q @ k.contiguous() * D ** -0.5
                later = torch.arange(length, device="cuda")[None, :] > place.repeat_interleave(group)[:, None]
                sc[later] = -math.inf
                w = torch.exp(sc - sc.max(1, keepdim=True).values)
                o = (w @ v.t().contiguous()) / w.sum(1, keepdim=True)
                out[at:at + n, h * group:(h + 1) * group] = o.view(n, group, D)
        at += n
    return [out]
