"""Measured cases of the operators around the attention call: rotary positions with several axes (with the norm of the
query and key heads), the FP8 preparation with them, and attention over packed sequences with grouped heads.

`run` computes a case in its plain form (elementary torch operations in 32 bits, angles in 64), or, where `own` is
true, through the package's public entry points.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
D = 128
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "open-vc-attention_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import open_vc_attn

    return open_vc_attn


# ---- the cases -------------------------------------------------------------------------------------------------


def _rotary(name, batch, s, hq, hk, axes, dtype, layout, freq, norm, start, fused):
    return dict(name=name, op="rotary", batch=batch, s=s, hq=hq, hk=hk, axes=axes, dtype=dtype, layout=layout, freq=freq,
                norm=norm, start=start, fused=fused)


def _prepare(name, s, h, axes, dtype, layout, freq, norm, start):
    return dict(name=name, op="prepare", s=s, h=h, axes=axes, dtype=dtype, layout=layout, freq=freq, norm=norm, start=start)


def _packed(name, hq, hk, q_lens, k_lens, causal, dtype, fused):
    return dict(name=name, op="packed", hq=hq, hk=hk, q_lens=q_lens, k_lens=k_lens, causal=causal, dtype=dtype, fused=fused)


def listed():
    return [
        # One new token of each of a few requests of a text model: q and k of a fused projection, far positions. Latency.
        _rotary("rotary-tokens", 1, 5, 32, 8, "128", "bf16", "half", "axis", True, 30000, True),
        # A batch of video clips at the batched path's benchmark shape, with the norm of the heads.
        _rotary("rotary-batch-8191", 4, 8191, 24, 24, "16,56,56", "fp16", "adjacent", "axis", True, 0, False),
        # One long video, a fourth of the headline workload's heads (one rank of a sharded job), no norm.
        _rotary("rotary-73397", 1, 73397, 14, 14, "44,42,42", "bf16", "adjacent", "axis", False, 0, False),
        # The smallest benchmark configuration of the FP8 path: latency.
        _prepare("prepare-1024", 1024, 2, "44,42,42", "bf16", "adjacent", "axis", False, 0),
        # The second benchmark configuration, sections of one set of frequencies over the three axes, norm.
        _prepare("prepare-32768", 32768, 8, "32,48,48", "fp16", "half", "head", True, 17),
        # One long video on one rank, an odd length, norm.
        _prepare("prepare-73397", 73397, 14, "44,42,42", "bf16", "adjacent", "axis", True, 0),
        # One short sequence, a key tile and one key more: latency.
        _packed("packed-129", 2, 2, "129", "129", False, "bf16", False),
        # Prompts of very different lengths in one batch, causal, grouped heads, slices of a fused projection.
        _packed("packed-prompts", 32, 8, "5000,3001,2048,777,129,1", "", True, "bf16", True),
        # Two clips packed, not causal, the batched path's head count and type.
        _packed("packed-clips", 24, 24, "8191,2730", "", False, "fp16", False),
        # One long sequence at the second benchmark configuration.
        _packed("packed-32768", 8, 8, "32768", "", False, "bf16", False),
        # One new token for each of sixteen requests whose keys are of very different lengths.
        _packed("packed-tokens", 32, 8, "1,1,1,1,1,1,1,1,1,1,1,1,1,1,1,1",
                "32768,20011,16384,12345,8192,8191,5000,4097,4096,3000,2048,1025,1000,512,129,1", True, "bf16", False),
        # Chunks of new tokens behind long prefixes, seven query heads to a key head.
        _packed("packed-chunks", 28, 4, "512,300,64,17", "16384,9000,30000,4113", True, "fp16", False),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5))))


def draw(rng):
    op = rng.choice(["rotary", "prepare", "packed", "packed", "packed"])
    dtype = rng.choice(["bf16", "fp16"])
    layout = rng.choice(["adjacent", "half"])
    axes = rng.choice(["128", "44,42,42", "16,56,56", "32,48,48", "64,64", "40,40,40"] if layout == "adjacent" else
                      ["128", "32,48,48", "44,42,42", "16,56,56", "64,64"])
    freq, norm = rng.choice(["axis", "head"]), rng.random() < 0.5
    start = rng.choice([0, 0, _log(rng, 1, 200000)])
    if op == "rotary":
        hq, hk = rng.choice([(32, 8), (24, 24), (14, 14), (7, 7), (28, 4), (16, 1), (56, 56), (1, 1)])
        batch = rng.choice([1, 1, 2, 3, 4])
        c = _rotary("", batch, _log(rng, 1, 73397 * 28 // ((hq + hk) * batch)), hq, hk, axes, dtype, layout, freq, norm, start,
                    rng.random() < 0.3)
    elif op == "prepare":
        h = rng.choice([1, 2, 3, 7, 8, 14])
        c = _prepare("", _log(rng, 1, 73397), h, axes, dtype, layout, freq, norm, start)
    else:
        hq, hk = rng.choice([(8, 8), (24, 24), (14, 14), (32, 8), (28, 4), (16, 1), (9, 3), (7, 7), (40, 8)])
        kind = rng.choice(["prompts", "pieces", "tokens", "chunks"])
        if kind == "tokens":
            b = _log(rng, 1, 32)
            most = min(32768, 6000000 // (hk * b))
            k = [_log(rng, 1, most) for _ in range(b)]
            q = [rng.choice([1, 1, 1, 2, 5]) for _ in range(b)]
            causal = rng.random() < 0.7
        elif kind == "chunks":
            b = _log(rng, 1, 6)
            q = [_log(rng, 1, 600) for _ in range(b)]
            most = max(2, min(32768, 2000000000 // (hq * b * max(q))))
            k = [_log(rng, 1, most) for _ in range(b)]
            causal = rng.random() < 0.7
        else:
            b = _log(rng, 1, 8)
            most = int(math.sqrt(2500000000 / (hq * b)))
            q = [_log(rng, 1, most) for _ in range(b)]
            k, causal = q, kind == "prompts"
            if b > 2 and rng.random() < 0.3:
                q[rng.randrange(b)] = 0
        ql, kl = ",".join(map(str, q)), ",".join(map(str, k))
        c = _packed("", hq, hk, ql, "" if ql == kl else kl, causal, dtype, kind == "prompts" and rng.random() < 0.5)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------


def _ints(text):
    return [int(x) for x in text.split(",")]


def _positions(s, n_axes, start):
    """One axis: consecutive positions. More: frames, rows and columns of a clip of 30 x 52 patches, in raster order, after
    `start` frames; a two-axis case leaves the frames out."""
    i = torch.arange(s, device=DEV)
    if n_axes == 1:
        p = (start + i)[:, None]
    else:
        p = torch.stack([start + i // 1560, i % 1560 // 52, i % 52], -1)[:, 3 - n_axes:]
    return p.to(torch.int32).contiguous()


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _split(g, t, heads, dtype, fused):
    """Tensors [*t, h, 128]: each its own, or slices of one fused projection."""
    if fused:
        x = _randn(g, *t, sum(heads), D).to(dtype)
        return list(x.split(heads, dim=-2))
    return [_randn(g, *t, h, D).to(dtype) for h in heads]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    st = dict(case)
    if case["op"] == "packed":
        q_lens = _ints(case["q_lens"])
        k_lens = _ints(case["k_lens"]) if case["k_lens"] else q_lens
        if case["fused"]:
            st["q"], st["k"], st["v"] = _split(g, [sum(q_lens)], [case["hq"], case["hk"], case["hk"]], dtype, True)
        else:
            st["q"] = _randn(g, sum(q_lens), case["hq"], D).to(dtype)
            st["k"], st["v"] = _split(g, [sum(k_lens)], [case["hk"]] * 2, dtype, False)
        cu = [torch.tensor([0] + x, device=DEV).cumsum(0).to(torch.int32) for x in (q_lens, k_lens)]
        st["cu_q"], st["cu_k"] = cu[0], cu[1] if case["k_lens"] else cu[0]
        st["max_q"], st["max_k"] = max(q_lens), max(k_lens)
        return st
    axes = _ints(case["axes"])
    if case["op"] == "rotary":
        st["q"], st["k"] = _split(g, [case["batch"], case["s"]], [case["hq"], case["hk"]], dtype, case["fused"])
    else:
        st["q"], st["k"], st["v"] = _split(g, [case["s"]], [case["h"]] * 3, dtype, False)
    st["positions"] = _positions(case["s"], len(axes), case["start"])
    st["qw"] = st["kw"] = None
    if case["norm"]:
        st["qw"], st["kw"] = [1 + 0.2 * _randn(g, D) for _ in range(2)]
    st["pair_axis"], st["frequency"] = _frequencies(axes, case["freq"])
    if own:
        st["plan"] = _package().rotary_plan(
            st["positions"], axes=tuple(axes), interleaved=case["layout"] == "adjacent", frequencies=case["freq"],
            q_weight=st["qw"], k_weight=st["kw"], eps=EPS)
    return st


def _frequencies(axes, freq):
    """For each rotated pair of channels its axis and its angle per position: 10000^(-2 i / d), i and d counted within the
    axis, or over all axes together."""
    total = sum(axes)
    axis = [a for a, d in enumerate(axes) for _ in range(d // 2)]
    if freq == "axis":
        f = [10000.0 ** (-2.0 * i / d) for d in axes for i in range(d // 2)]
    else:
        f = [10000.0 ** (-2.0 * i / total) for i in range(total // 2)]
    return torch.tensor(axis, device=DEV), torch.tensor(f, dtype=torch.float64, device=DEV)


# ---- the plain forms -------------------------------------------------------------------------------------------


def _plain_rotate(x, w, st):
    """x / rms(x) * w, then each pair (a, b) of channels turned by its angle; 32 bits, angles in 64."""
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    angle = st["positions"].double()[:, st["pair_axis"]] * st["frequency"]
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    n = 2 * angle.shape[-1]
    if st["layout"] == "adjacent":
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, x[..., n:]], -1) if n < D else turned


def _plain_codes(x, amax):
    return (x * (448.0 / amax)).clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_blocks(x):
    """E4M3 codes with one scale for each head and 128 tokens, and the scales [1, H, blocks]."""
    s, h, _ = x.shape
    blocks = -(-s // 128)
    pad = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, blocks * 128 - s)).view(blocks, 128, h, D)
    amax = pad.abs().amax((1, 3), keepdim=True).clamp_min(1e-12)
    return _plain_codes(pad, amax).view(-1, h, D)[:s], (amax / 448.0).view(1, blocks, h).transpose(1, 2).contiguous()


def _plain_prepare(st):
    q8, qs = _plain_blocks(_plain_rotate(st["q"], st["qw"], st))
    k8, ks = _plain_blocks(_plain_rotate(st["k"], st["kw"], st))
    v = st["v"].float()
    amax = v.abs().amax((0, 2)).clamp_min(1e-12)
    return {"q": q8, "k": k8, "v": _plain_codes(v, amax[:, None]), "q_descale": qs, "k_descale": ks,
            "v_descale": (amax / 448.0)[None]}


def _rows(cu, most):
    """For a padded [B, most] layout of packed rows: which places hold a row, and which row."""
    lens = (cu[1:] - cu[:-1])[:, None]
    i = torch.arange(most, device=DEV)[None]
    return i < lens, (cu[:-1, None] + i.minimum((lens - 1).clamp_min(0))).long().clamp_max(int(1e18))


def _plain_packed(st):
    hq, hk = st["hq"], st["hk"]
    has_q, at_q = _rows(st["cu_q"], st["max_q"])
    has_k, at_k = _rows(st["cu_k"], st["max_k"])
    at_q, at_k = at_q.clamp_max(st["q"].shape[0] - 1), at_k.clamp_max(st["k"].shape[0] - 1)
    b, lq, lk, g = has_q.shape[0], st["max_q"], st["max_k"], hq // hk
    q = (st["q"][at_q].float() * D ** -0.5).view(b, lq, hk, g, D).permute(0, 2, 3, 1, 4).reshape(b, hk, g * lq, D)
    k, v = st["k"][at_k].float().permute(0, 2, 3, 1), st["v"][at_k].float().transpose(1, 2)
    scores = (q @ k).view(b, hk, g, lq, lk)
    hidden = ~has_k[:, None, :]
    if st["causal"]:
        # the last new token sees every key: row r of a sequence sees the keys up to r + (keys - rows)
        more = ((st["cu_k"][1:] - st["cu_k"][:-1]) - (st["cu_q"][1:] - st["cu_q"][:-1]))[:, None, None]
        i, j = torch.arange(lq, device=DEV)[None, :, None], torch.arange(lk, device=DEV)[None, None]
        hidden = hidden | (j > i + more)
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(b, hk, g * lq, lk) @ v).view(b, hk, g, lq, D)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, lq, hq, D)[has_q].to(st["q"].dtype)
    return out, lse.permute(0, 3, 1, 2).reshape(b, lq, hq)[has_q].t().contiguous()


def run(st):
    if own:
        ovc = _package()
        if st["op"] == "rotary":
            return ovc.rotary_qk(st["q"], st["k"], st["plan"])
        if st["op"] == "packed":
            return ovc.attention_packed(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], causal=st["causal"], return_lse=True)
        fuse = ovc.prepare_fp8_fused if st["s"] >= 32768 else ovc.prepare_fp8
        p = fuse(st["q"], st["k"], st["v"], rotary=st["plan"])
        blocks = p.k_descale.shape[-1]  # the fused preparation rounds the query blocks up to an even count
        return {"q": p.q, "k": p.k, "v": p.v, "q_descale": p.q_descale[..., :blocks], "k_descale": p.k_descale,
                "v_descale": p.v_descale}
    if st["op"] == "rotary":
        return tuple(_plain_rotate(st[n], st[n + "w"], st).to(st[n].dtype) for n in "qk")
    return _plain_packed(st) if st["op"] == "packed" else _plain_prepare(st)


# ---- what a case cannot do without -----------------------------------------------------------------------------


def work(case):
    if case["op"] == "rotary":
        x = case["batch"] * case["s"] * (case["hq"] + case["hk"]) * D
        return {"bytes": 4 * x + 4 * case["s"] * len(_ints(case["axes"])), "flops": (3 + 4 * case["norm"]) * x}
    if case["op"] == "prepare":
        x = case["s"] * case["h"] * D
        return {"bytes": 9 * x + 4 * case["s"] * len(_ints(case["axes"])) + 8 * case["h"] * -(-case["s"] // 128),
                "flops": (2 * (6 + 4 * case["norm"]) + 3) * x}
    q = _ints(case["q_lens"])
    k = _ints(case["k_lens"]) if case["k_lens"] else q
    seen = 0
    for a, b in zip(q, k):
        if not case["causal"]:
            seen += a * b
        else:  # rows r = 0 .. a-1 see r + 1 + b - a keys, none where that is negative
            full, first = min(a, b), max(0, b - a)
            seen += full * first + full * (full + 1) // 2
    rows = sum(q) * case["hq"]
    return {"bytes": 4 * rows * D + 4 * rows + 4 * sum(k) * case["hk"] * D, "flops": 4 * D * case["hq"] * seen}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------


def _exact_rotate(x, w, st, axes):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
    total, at, angles = sum(axes), 0, []
    for a, d in enumerate(axes):
        i = torch.arange(d // 2, dtype=torch.float64, device=DEV)
        power = i / d if st["freq"] == "axis" else (at + i) / total
        angles.append(torch.outer(st["positions"][:, a].double(), torch.exp(-2 * power * math.log(10000.0))))
        at += d // 2
    angle = torch.cat(angles, -1)[:, None]
    turn = torch.polar(torch.ones_like(angle), angle)
    y = x.clone()
    if st["layout"] == "adjacent":
        z = torch.complex(x[..., 0:total:2].contiguous(), x[..., 1:total:2].contiguous()) * turn
        y[..., 0:total:2], y[..., 1:total:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :total // 2].contiguous(), x[..., total // 2:].contiguous()) * turn
        y[..., :total // 2], y[..., total // 2:] = z.real, z.imag
    return y


def _exact_blocks(x):
    codes, scales = torch.empty_like(x), []
    for at in range(0, x.shape[0], 128):
        block = x[at:at + 128]
        scale = block.abs().amax((0, 2)).clamp_min(1e-12) / 448
        codes[at:at + 128] = block / scale[:, None]
        scales.append(scale)
    return codes, torch.stack(scales, -1)[None]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "packed":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
        lse = torch.full((case["hq"], st["q"].shape[0]), -math.inf, dtype=torch.float64, device=DEV)
        cu_q, cu_k, g = st["cu_q"].tolist(), st["cu_k"].tolist(), case["hq"] // case["hk"]
        for b in range(len(cu_q) - 1):
            q0, q1, k0, k1 = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
            for h in range(case["hk"]):
                k, v = st["k"][k0:k1, h].double(), st["v"][k0:k1, h].double()
                for r0 in range(q0, q1, 1024):
                    r1 = min(q1, r0 + 1024)
                    heads = slice(h * g, h * g + g)
                    s = torch.einsum("rgd,kd->rgk", st["q"][r0:r1, heads].double(), k) / math.sqrt(D)
                    if case["causal"]:
                        last = torch.arange(r0, r1, device=DEV) - q1 + k1 - k0
                        s = torch.where(torch.arange(k1 - k0, device=DEV) <= last[:, None, None], s, -math.inf)
                    if k1 > k0:
                        lse[heads, r0:r1] = torch.logsumexp(s, -1).t()
                        p = torch.nan_to_num(torch.softmax(s, -1))
                        out[r0:r1, heads] = torch.einsum("rgk,kd->rgd", p, v)
        return out, lse
    axes = _ints(case["axes"])
    q, k = _exact_rotate(st["q"], st["qw"], st, axes), _exact_rotate(st["k"], st["kw"], st, axes)
    if case["op"] == "rotary":
        return q, k
    (q, qs), (k, ks) = _exact_blocks(q), _exact_blocks(k)
    v = st["v"].double()
    vs = v.abs().amax((0, 2)).clamp_min(1e-12) / 448
    return {"q": q, "k": k, "v": v / vs[:, None], "q_descale": qs, "k_descale": ks, "v_descale": vs[None]}
