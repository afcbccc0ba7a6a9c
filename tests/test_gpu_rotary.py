"""Rotary positions with several axes, alone and inside the FP8 preparation, against the formula in 64 bits.

Tolerances.  Every output is one rounding of a float32 value.  For that value each factor has a few float32 roundings: the
norm (a sum of 128 squares, eight by eight and then four pairwise steps: at most 12 roundings of the sum, half of that after
the root, rsqrtf 2 ulp, two products) under 12 * 2^-24 relative; cos and sin within 2^-24 * pi of the angle's rounding plus 2
ulp of sincospif, under 6 * 2^-24 absolute; the two products and the sum 3 * 2^-24.  So |error| <= 24 * 2^-24 * hypot(a, b) * |w|
max, for the pair (a, b) normalised, plus half a step of the output type (2^-8 bf16, 2^-11 fp16 relative to the value).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from gpu_util import DEV  # noqa: E402

F32 = 24 * 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _ovc():
    import open_vc_attn

    return open_vc_attn


def formula(x, positions, axes, interleaved=True, frequencies="axis", theta=10000.0, weight=None, eps=1e-6):
    """([.., S, H, 128] float64 result, the length of each channel's pair, which bounds its float32 error)."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    total, first, angles = sum(axes), 0, []
    for a, d in enumerate(axes):
        i = torch.arange(d // 2, device=x.device, dtype=torch.float64)
        e = 2 * i / d if frequencies == "axis" else 2 * (first + i) / total
        angles.append(positions[..., a].double()[..., None] * theta ** -e)
        first += d // 2
    t = torch.cat(angles, -1)[..., None, :]
    i = torch.arange(total // 2, device=x.device)
    at, to = (2 * i, 2 * i + 1) if interleaved else (i, i + 64)
    y, size = x.clone(), x.abs()
    a, b = x[..., at], x[..., to]
    y[..., at], y[..., to] = a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()
    size[..., at] = size[..., to] = torch.hypot(a, b)
    return y, size


def close(got, want, size):
    off = (got.double() - want).abs()
    limit = F32 * size + HALF_STEP[got.dtype] * want.abs() + (2.0 ** -24 if got.dtype == torch.float16 else 0.0)
    limit = limit * (1 + 2.0 ** -7)  # the half step is relative to the value before it was rounded, off by the first term
    assert bool((off <= limit).all()), float((off - limit).max())


def inputs(shape_q, shape_k, seed, dtype):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, k = [torch.randn(s, generator=g, device=DEV).to(dtype) for s in (shape_q, shape_k)]
    return q, k, [1 + 0.25 * torch.randn(128, generator=g, device=DEV) for _ in range(2)]


CASES = [
    # batch, tokens, q heads, k heads, axes, interleaved, frequencies, norm, type
    (1, 1, 1, 1, (128,), False, "axis", True, torch.bfloat16),
    (1, 1, 56, 56, (44, 42, 42), True, "axis", False, torch.float16),
    (1, 17, 32, 8, (128,), False, "axis", True, torch.bfloat16),
    (2, 129, 3, 1, (16, 56, 56), True, "axis", True, torch.float16),
    (3, 77, 7, 7, (32, 48, 48), False, "head", True, torch.bfloat16),
    (1, 1000, 28, 4, (40, 40, 40), True, "head", False, torch.bfloat16),
    (1, 9001, 2, 2, (2, 2, 2, 2), True, "axis", True, torch.float16),
    (2, 5000, 5, 9, (64, 64), False, "axis", False, torch.bfloat16),
]


@pytest.mark.parametrize("batch,s,hq,hk,axes,interleaved,frequencies,norm,dtype", CASES)
@pytest.mark.parametrize("kind", ["int32", "int64", "float32", "per item"])
def test_rotation_matches_the_formula(batch, s, hq, hk, axes, interleaved, frequencies, norm, dtype, kind):
    ovc = _ovc()
    q, k, (qw, kw) = inputs((batch, s, hq, 128), (batch, s, hk, 128), s + hq, dtype)
    g = torch.Generator(device=DEV).manual_seed(5)
    lead = (batch, s) if kind == "per item" else (s,)
    positions = torch.randint(0, 200000, (*lead, len(axes)), generator=g, device=DEV)
    if kind == "float32":
        positions = positions.float() / 7.0
    elif kind != "int64":
        positions = positions.int()
    plan = ovc.rotary_plan(positions, axes=axes, interleaved=interleaved, frequencies=frequencies,
                           q_weight=qw if norm else None, k_weight=kw if norm else None)
    got = ovc.rotary_qk(q, k, plan)
    for x, y, w in zip((q, k), got, (qw, kw)):
        assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
        close(y, *formula(x, positions, axes, interleaved, frequencies, weight=w if norm else None))
    again = ovc.rotary_qk(q, k, plan)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    if batch == 1 and kind != "per item":  # a 3-D call is the same sequence
        assert all(torch.equal(a[0], b) for a, b in zip(got, ovc.rotary_qk(q[0], k[0], plan)))


@pytest.mark.parametrize("s", [1, 40, 6000])
def test_slices_of_a_fused_projection_and_other_strides(s):
    ovc = _ovc()
    g = torch.Generator(device=DEV).manual_seed(s)
    qkv = torch.randn(2, s, 12, 128, generator=g, device=DEV).to(torch.bfloat16)
    q, k = qkv[:, :, :6], qkv[:, :, 6:9]
    positions = torch.arange(s, device=DEV)[:, None]
    plan = ovc.rotary_plan(positions, axes=(128,))
    dense = ovc.rotary_qk(q.contiguous(), k.contiguous(), plan)
    assert all(torch.equal(a, b) for a, b in zip(ovc.rotary_qk(q, k, plan), dense))
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]  # [B,H,S,128] storage
    assert all(torch.equal(a, b) for a, b in zip(ovc.rotary_qk(*heads_first, plan), dense))
    odd = torch.randn(2, s, 9, 129, generator=g, device=DEV).to(torch.bfloat16)[..., 1:]  # rows off the 16-byte grid: copied
    assert all(torch.equal(a, b) for a, b in zip(ovc.rotary_qk(odd[:, :, :6], odd[:, :, 6:], plan),
                                                 ovc.rotary_qk(odd[:, :, :6].contiguous(), odd[:, :, 6:].contiguous(), plan)))
    one = q[:, :, :1].expand(2, s, 6, 128)  # one head shown six times
    assert torch.equal(ovc.rotary_qk(one, k, plan)[0], ovc.rotary_qk(one.contiguous(), k, plan)[0])


def test_special_values():
    ovc = _ovc()
    plan = ovc.rotary_plan(torch.zeros(4, 3, device=DEV, dtype=torch.int32), q_weight=torch.ones(128, device=DEV))
    x = torch.zeros(4, 1, 128, device=DEV, dtype=torch.bfloat16)
    x[1, 0, 5] = math.inf
    x[2, 0, 6] = math.nan
    x[3] = 3.0e38
    q, k = ovc.rotary_qk(x, x, plan)
    assert not q[0].any()  # 0 / sqrt(eps)
    assert q[1:3].isnan().any(-1).all()
    # a head that is not normalised and sits at position zero comes back bit for bit (a pair with an infinity has 0 * inf)
    assert torch.equal(k[0], x[0]) and torch.equal(k[3], x[3])
    text = ovc.grid_positions(2, 3, 4, text=5, start=(1, 0, 0), device=DEV)
    assert text.shape == (29, 3) and not text[:5].any() and text[5].tolist() == [1, 0, 0] and text[-1].tolist() == [2, 2, 3]


@pytest.mark.parametrize("batch,s,h,axes,interleaved,frequencies,norm,dtype", [
    (1, 1, 1, (128,), False, "axis", True, torch.bfloat16),
    (1, 127, 2, (44, 42, 42), True, "axis", True, torch.bfloat16),
    (1, 129, 3, (32, 48, 48), False, "head", False, torch.float16),
    (3, 300, 5, (16, 56, 56), True, "axis", True, torch.float16),
    (1, 5000, 14, (40, 40, 40), True, "head", True, torch.bfloat16),
    (1, 33001, 3, (44, 42, 42), True, "axis", True, torch.bfloat16),  # the fused preparation
])
def test_preparation_rotates_what_it_quantises(batch, s, h, axes, interleaved, frequencies, norm, dtype):
    """Codes: E4M3 of value / descale: half a step (2^-4 relative, 2^-10 below the normal range) around the exact value, plus
    the float32 error of the value (F32 of the pair's length) and of the scale.  Descales: the exact block maximum / 448,
    within the float32 error of the largest value and of one division (div.full: 2 ulp)."""
    ovc = _ovc()
    shape = (batch, s, h, 128) if batch > 1 else (s, h, 128)
    q, k, (qw, kw) = inputs(shape, shape, s, dtype)
    v = torch.randn(shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
    positions = torch.randint(0, 5000, (s, len(axes)), device=DEV, dtype=torch.int32, generator=torch.Generator(device=DEV).manual_seed(2))
    plan = ovc.rotary_plan(positions, axes=axes, interleaved=interleaved, frequencies=frequencies,
                           q_weight=qw if norm else None, k_weight=kw if norm else None)
    fused = s >= 32768
    got = (ovc.prepare_fp8_fused if fused else ovc.prepare_fp8)(q, k, v, rotary=plan)
    plain = (ovc.prepare_fp8_fused if fused else ovc.prepare_fp8)(q, k, v)
    blocks = -(-s // 128)
    assert torch.equal(got.v.float(), plain.v.float()) and torch.equal(got.v_descale, plain.v_descale)
    assert got.q_descale.shape == plain.q_descale.shape and got.k_descale.shape == plain.k_descale.shape
    if got.q_descale.shape[-1] > blocks:
        assert bool((got.q_descale[..., blocks:] == 1.0).all())
    for x, w, codes, descale in ((q, qw, got.q, got.q_descale), (k, kw, got.k, got.k_descale)):
        want, size = formula(x, positions, axes, interleaved, frequencies, weight=w if norm else None)
        want, size = [t.view(batch, s, h, 128) for t in (want, size)]
        pad = torch.nn.functional.pad(want.abs(), (0, 0, 0, 0, 0, blocks * 128 - s)).view(batch, blocks, 128, h, 128)
        top = pad.amax((2, 4)).clamp_min(1e-12).transpose(1, 2)  # [B,H,blocks]
        longest = torch.nn.functional.pad(size, (0, 0, 0, 0, 0, blocks * 128 - s)).view(batch, blocks, 128, h, 128).amax((2, 4)).transpose(1, 2)
        d = descale.double()[..., :blocks]
        assert bool(((d * 448 - top).abs() <= F32 * longest + 4 * 2.0 ** -24 * top).all())
        per_token = d.transpose(1, 2).repeat_interleave(128, 1)[:, :s, :, None]
        value, off = want / per_token, F32 * size / per_token + 4 * 2.0 ** -24 * (want / per_token).abs()
        limit = (value.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) + 1.1 * off
        assert bool(((codes.double().view(batch, s, h, 128) - value).abs() <= limit).all())


@pytest.mark.parametrize("shape", [(777, 3), (2, 400, 4), (32769, 2)])
def test_attention_rotates_as_a_call_of_its_own_does(shape):
    """attention(rotary=plan) is attention_fp8 of the rotated preparation, bit for bit, and agrees with attention of
    separately rotated Q and K: those were rounded to 16 bits in between, so a few codes differ by a step."""
    ovc = _ovc()
    shape = (*shape, 128)
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = [torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16) for _ in range(3)]
    s = shape[-3]
    plan = ovc.rotary_plan(torch.stack([torch.arange(s, device=DEV)] * 3, -1), q_weight=torch.ones(128, device=DEV))
    out = ovc.attention(q, k, v, rotary=plan)
    fused = s >= 32768
    prepared = (ovc.prepare_fp8_fused if fused else ovc.prepare_fp8)(q, k, v, rotary=plan)
    assert torch.equal(out, ovc.attention_fp8(prepared))
    apart = ovc.attention(*ovc.rotary_qk(q, k, plan), v)
    assert float((out.float() - apart.float()).norm() / apart.float().norm()) < 2.0 ** -4 * 2  # two E4M3 half steps, Q and K


def test_graph_capture_side_stream_and_concurrent_calls():
    ovc = _ovc()
    q, k, _ = inputs((500, 6, 128), (500, 2, 128), 4, torch.bfloat16)
    positions = torch.arange(500, device=DEV)[:, None]
    plan = ovc.rotary_plan(positions, axes=(128,))
    want = ovc.rotary_qk(q, k, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ovc.rotary_qk(q, k, plan)
        same = ovc.rotary_qk(q, k, plan)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, other, same))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ovc.rotary_qk(q, k, plan)
    fresh = torch.randn_like(q.float()).to(q.dtype)
    q.copy_(fresh)
    positions.add_(3)  # the plan refers to the caller's tensor
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, ovc.rotary_qk(q, k, plan)))


def test_refusals_on_the_device():
    ovc = _ovc()
    q, k, _ = inputs((8, 2, 128), (8, 2, 128), 1, torch.bfloat16)
    plan = ovc.rotary_plan(torch.zeros(8, 3, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="7"):
        ovc.rotary_qk(q[:7], k[:7], plan)
    with pytest.raises(ValueError, match="same tokens"):
        ovc.rotary_qk(q, k[:7], plan)
    with pytest.raises(ValueError, match="matching dtypes"):
        ovc.rotary_qk(q, k.half(), plan)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        ovc.rotary_qk(q.float(), k.float(), plan)
    with pytest.raises(TypeError, match="rotary_plan"):
        ovc.rotary_qk(q, k, object())
    with pytest.raises(TypeError, match="rotary_plan"):
        ovc.attention(q, k, k, rotary=torch.zeros(8, 3, device=DEV))
    with pytest.raises(ValueError, match="same tokens"):
        ovc.attention(q, k[:5], k[:5], rotary=plan)
    with pytest.raises(ValueError, match="detach"):
        ovc.rotary_qk(q.clone().requires_grad_(), k, plan)
    with pytest.raises(ValueError, match="axes"):
        ovc.rotary_plan(torch.zeros(8, 2, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="q_weight"):
        ovc.rotary_plan(torch.zeros(8, 3, device=DEV, dtype=torch.int32), q_weight=torch.ones(64, device=DEV))
    empty = ovc.rotary_qk(q[:0], k[:0], ovc.rotary_plan(torch.zeros(0, 3, device=DEV, dtype=torch.int32)))
    assert empty[0].shape == (0, 2, 128)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_plan_keeps_its_weights(dtype):
    ovc = _ovc()
    q, k, _ = inputs((40, 2, 128), (40, 2, 128), 1, torch.bfloat16)
    weight = torch.rand(256, device=DEV).to(dtype)[::2]
    plan = ovc.rotary_plan(torch.arange(40, device=DEV)[:, None], axes=(128,), q_weight=weight, k_weight=weight)
    want = ovc.rotary_qk(q, k, plan)
    weight.zero_()
    assert all(torch.equal(a, b) for a, b in zip(want, ovc.rotary_qk(q, k, plan)))


@pytest.mark.parametrize("s,h", [(500, 3), (32769, 2)])
def test_preparation_captured_repeated_and_on_two_streams(s, h):
    """The kernels of a preparation start before the ones in front of them have ended; back to back on one stream, in a
    replayed graph and on two streams at once they give what a call by itself gives."""
    ovc = _ovc()
    prepare = ovc.prepare_fp8_fused if s >= 32768 else ovc.prepare_fp8
    plan = ovc.rotary_plan(torch.arange(s, device=DEV)[:, None], axes=(128,))
    sets = []
    for i in range(4):
        q, k, _ = inputs((s, h, 128), (s, h, 128), 20 + i, torch.bfloat16)
        sets.append((q, k, (k.float() * (i + 1) - 0.5 * q.float()).to(q.dtype)))

    def values(p):
        return [t.clone().view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.clone()
                for t in (p.q, p.k, p.v, p.q_descale, p.k_descale, p.v_descale)]

    want = []
    for qkv in sets:
        want.append(values(prepare(*qkv, rotary=plan)))
        torch.cuda.synchronize()
    assert not torch.equal(want[0][5], want[1][5])

    def check(got):
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(values(g), w))

    check([prepare(*qkv, rotary=plan) for qkv in sets])
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for i, qkv in enumerate(sets):
        with torch.cuda.stream(streams[i % 2]):
            got.append(prepare(*qkv, rotary=plan))
    check(got)
    static = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = prepare(*static, rotary=plan)
    for qkv, w in zip(sets, want):
        for to, t in zip(static, qkv):
            to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(values(captured), w))


@pytest.mark.parametrize("s,fused", [(1, False), (300, False), (32768, True), (32900, True)])
def test_preparation_hands_its_bounds_on(s, fused):
    ovc = _ovc()
    q, k, _ = inputs((s, 2, 128), (s, 2, 128), 9, torch.float16)
    plan = ovc.rotary_plan(torch.arange(s, device=DEV)[:, None], axes=(128,))
    for first in (q, q[None]):
        second = k.reshape(first.shape)
        prepared = (ovc.prepare_fp8_fused if fused else ovc.prepare_fp8)(first, second, second, rotary=plan)
        layout = prepared.layout
        assert layout["cu_seqlens_q"].tolist() == layout["cu_seqlens_k"].tolist() == [0, s]
        assert layout["max_seqlen_q"] == layout["max_seqlen_k"] == s
    if fused:
        mine = torch.tensor([0, s], device=DEV, dtype=torch.int32)
        assert ovc.prepare_fp8_fused(q, k, k, cu_seqlens=mine, rotary=plan).layout["cu_seqlens_q"] is mine
    batch = ovc.prepare_fp8(torch.stack([q, k]), torch.stack([k, q]), torch.stack([k, k]), rotary=plan)
    assert batch.layout == {}


def turned(x, positions, turns, half=False):
    """``formula`` for 64 frequencies in turns per position, of any size and sign, on one axis: the product is exact in whole
    numbers of 2^-40 turns for the values used here, so its fraction is, too."""
    t = (positions.double()[..., 0, None] * turns).remainder(1.0) * (2.0 * math.pi)
    t, i = t[:, None], torch.arange(64, device=x.device)
    at, to = (i, i + 64) if half else (2 * i, 2 * i + 1)
    y, size = x.double(), x.double().abs()
    a, b = x.double()[..., at], x.double()[..., to]
    y[..., at], y[..., to] = a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()
    size[..., at] = size[..., to] = torch.hypot(a, b)
    return y, size


FRACTIONAL = [0.5, 2.25, -0.5, -3.75, 0.0, 1.0, 2.0 ** -12 * 5, 4097.125, -(2.0 ** 20) + 0.5, 1.5 * 2.0 ** 30]


@pytest.mark.parametrize("theta", [0.05, 0.1, 0.9, 1e-6, 10000.0])
@pytest.mark.parametrize("interleaved", [False, True])
def test_fractional_positions_and_fast_frequencies(theta, interleaved):
    """Small thetas turn by more than a whole turn per position, of which a fractional position takes a fraction."""
    ovc = _ovc()
    positions = torch.tensor([p for p in FRACTIONAL if abs(p) < 5], device=DEV)[:, None]
    s = positions.shape[0]
    q, k, _ = inputs((s, 3, 128), (s, 2, 128), 12, torch.bfloat16)
    got = ovc.rotary_qk(q, k, ovc.rotary_plan(positions, axes=(128,), theta=theta, interleaved=interleaved))
    for x, y in zip((q, k), got):
        # (below 2^20 turns in all, whose products and frequencies in 64 bits are off by 2^-31 turns at most)
        close(y, *formula(x, positions, (128,), interleaved, theta=theta))


@pytest.mark.parametrize("kind", [torch.float32, torch.int32, torch.int64])
@pytest.mark.parametrize("half", [False, True])
def test_frequencies_of_any_size_and_sign(kind, half):
    """The C entry takes frequencies of either sign; the plan's own are replaced by some that are exact in 2^-20 turns."""
    ovc = _ovc()
    plan_positions = torch.tensor(FRACTIONAL, device=DEV)[:, None].to(kind)
    s = len(FRACTIONAL)
    plan = ovc.rotary_plan(plan_positions, axes=(128,), interleaved=not half)
    values = [0.0, 0.25, -0.25, 1.0, -1.0, 3.0, -3.0, 1.25, -1.25, 2.0 ** -20, -(2.0 ** -20), 1023.0 + 2.0 ** -20, -1023.0 - 2.0 ** -20]
    turns = [values[i % len(values)] for i in range(64)]
    plan.turns[:] = turns
    q, k, _ = inputs((s, 3, 128), (s, 2, 128), 13, torch.float16)
    for x, y in zip((q, k), ovc.rotary_qk(q, k, plan)):
        close(y, *turned(x, plan_positions, torch.tensor(turns, device=DEV, dtype=torch.float64), half))
    prepared = ovc.prepare_fp8(q[:, :2].contiguous(), k, k, rotary=plan)
    want, size = turned(k, plan_positions, torch.tensor(turns, device=DEV, dtype=torch.float64), half)
    d = prepared.k_descale.double()[0, :, 0][None, :, None]
    limit = (want / d).abs().mul(2.0 ** -4).clamp_min(2.0 ** -10) + 1.1 * (F32 * size / d + 4 * 2.0 ** -24 * (want / d).abs())
    assert bool(((prepared.k.double() - want / d).abs() <= limit).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("axes", [(40, 40, 40), (2, 2, 2), (4, 2, 120)])
@pytest.mark.parametrize("weighted", ["none", "q", "k"])
def test_channels_without_an_axis_stay_as_they_are(dtype, axes, weighted):
    """Zeros of either sign, infinities and NaN beside each other: the tensors that are not normalised keep every bit."""
    ovc = _ovc()
    s, total = 70, sum(axes)
    q, k, (qw, kw) = inputs((s, 9, 128), (s, 3, 128), total, dtype)
    special = torch.tensor([math.inf, 1.5, -0.0, math.nan, 2.0, -math.inf, -0.0, -3.0, 0.0, -0.0], device=DEV, dtype=dtype)
    rest = 128 - total
    if rest:
        pick = torch.randint(0, 10, (s, 3, rest), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
        q[:, :3, total:], k[..., total:] = special[pick], special[pick.flip(-1)]
    positions = torch.randint(0, 5000, (s, 3), device=DEV, dtype=torch.int32, generator=torch.Generator(device=DEV).manual_seed(2))
    plan = ovc.rotary_plan(positions, axes=axes, q_weight=qw if weighted == "q" else None, k_weight=kw if weighted == "k" else None)
    for name, x, y in zip("qk", (q, k), ovc.rotary_qk(q, k, plan)):
        if name != weighted:
            kept = [t[..., total:].contiguous().view(torch.int16) for t in (x, y)]
            nan = x[..., total:].isnan()
            assert torch.equal(kept[0][~nan], kept[1][~nan]) and torch.equal(nan, y[..., total:].isnan())
        finite = torch.isfinite(x).all(-1) if name == weighted else torch.ones(x.shape[:2], dtype=torch.bool, device=DEV)
        want, size = formula(x, positions, axes, weight=qw if weighted == "q" else kw if weighted == "k" else None) if name == weighted \
            else formula(x, positions, axes)
        close(y[finite][..., :total], want[finite][..., :total], size[finite][..., :total])


@pytest.mark.parametrize("half", [False, True])
def test_single_pairs_that_do_not_turn(half):
    """Frequencies of zero anywhere among the pairs, in either layout, at the C entry."""
    ovc = _ovc()
    plan = ovc.rotary_plan(torch.arange(50, device=DEV)[:, None], axes=(128,), interleaved=not half)
    turns = [0.0 if i % 3 == 0 or i in (7, 62) else 2.0 ** -(i % 11) for i in range(64)]
    plan.turns[:] = turns
    q, k, _ = inputs((50, 2, 128), (50, 5, 128), 3, torch.bfloat16)
    still = torch.tensor([i for i, t in enumerate(turns) if t == 0.0], device=DEV)
    at, to = (still, still + 64) if half else (2 * still, 2 * still + 1)
    q[:, 0, at], k[:, 1, to] = math.inf, -math.inf
    for x, y in zip((q, k), ovc.rotary_qk(q, k, plan)):
        assert torch.equal(x[..., at], y[..., at]) and torch.equal(x[..., to], y[..., to])
        clean = x.masked_fill(torch.isinf(x), 0.0)
        want, size = turned(clean, torch.arange(50, device=DEV)[:, None], torch.tensor(turns, device=DEV, dtype=torch.float64), half)
        moved = torch.tensor([c for c in range(128) if c not in set(at.tolist() + to.tolist())], device=DEV)
        close(y[..., moved], want[..., moved], size[..., moved])


@pytest.mark.parametrize("weighted", [False, True])
def test_preparation_keeps_channels_without_an_axis(weighted):
    """A NaN takes no part in its block's scale; the channel beside it, not turned, has the code of its own value."""
    from open_vc_attn.quantization import fp8_quantize_per_block

    ovc = _ovc()
    q, k, (qw, _) = inputs((300, 2, 128), (300, 2, 128), 8, torch.bfloat16)
    plan = ovc.rotary_plan(torch.zeros(300, 3, device=DEV, dtype=torch.int32), axes=(40, 40, 40), q_weight=qw if weighted else None)
    k[::7, :, 124] = math.nan
    got = ovc.prepare_fp8(q, k, k, rotary=plan)
    want, descale = fp8_quantize_per_block(k, block_l=128)
    keep = [c for c in range(128) if c != 124]
    assert torch.equal(got.k_descale, descale)
    assert torch.equal(got.k[..., keep].view(torch.uint8), want[0][..., keep].view(torch.uint8))  # (the quantiser's output is batched)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("axes,interleaved", [((44, 42, 42), True), ((128,), False), ((40, 40, 40), True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_of_values_that_are_not_finite(bad, axes, interleaved, dtype):
    """At position zero a rotation without norm leaves 16-bit values that rotary_qk rounds to themselves (and NaN, where zero
    times an infinity is added), so the preparation has the codes and scales of the quantiser on rotary_qk's output, but NaN
    for what is not finite, where that has -448."""
    from open_vc_attn.quantization import fp8_quantize_per_block

    ovc = _ovc()
    q, k, _ = inputs((700, 2, 128), (700, 2, 128), 19, dtype)
    q[130, 1, 3], q[131, :, 127], q[5, 0, 64] = bad, bad, bad
    k[300:400], k[699, 1, 121] = bad, bad
    plan = ovc.rotary_plan(torch.zeros(700, len(axes), device=DEV, dtype=torch.int32), axes=axes, interleaved=interleaved)
    got = ovc.prepare_fp8(q, k, k, rotary=plan)
    for x, codes, descale in zip(ovc.rotary_qk(q, k, plan), (got.q, got.k), (got.q_descale, got.k_descale)):
        want, want_descale = fp8_quantize_per_block(x, block_l=128)
        assert torch.equal(descale, want_descale)
        odd = ~torch.isfinite(x)
        assert bool(odd.any()) and bool((want[0].float()[odd].abs() == 448).all())
        assert bool(codes.float()[odd].isnan().all()) and torch.equal(codes.view(torch.uint8)[~odd], want[0].view(torch.uint8)[~odd])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_codes_of_normalised_heads_that_are_not_finite(bad):
    """Such a head has NaN (an infinity over an infinity) and zeros; other heads keep their codes, the block its scale."""
    ovc = _ovc()
    q, k, (qw, kw) = inputs((200, 3, 128), (200, 3, 128), 20, torch.bfloat16)
    positions = torch.arange(200, device=DEV)[:, None]
    plan = ovc.rotary_plan(positions, axes=(128,), q_weight=qw, k_weight=kw)
    q[7, 1] = 0.0
    clean = ovc.prepare_fp8(q, k, k, rotary=plan)
    q[7, 1, 10] = bad
    got = ovc.prepare_fp8(q, k, k, rotary=plan)
    codes, was = got.q.view(torch.uint8), clean.q.view(torch.uint8)
    assert torch.equal(got.q_descale, clean.q_descale) and torch.equal(got.k.view(torch.uint8), clean.k.view(torch.uint8))
    rotated = ovc.rotary_qk(q, k, plan)[0]
    nan = rotated.isnan()
    assert bool(nan[7, 1, 10]) and int(nan.any(-1).sum()) == 1
    assert torch.equal(got.q.float().isnan(), nan)
    others = torch.ones(200, 3, dtype=torch.bool, device=DEV)
    others[7, 1] = False
    assert torch.equal(codes[others], was[others])
    assert bool((codes[7, 1][~nan[7, 1]] & 0x7F == 0).all())


@pytest.mark.parametrize("per_item", [False, True])
def test_a_batch_of_many_short_sequences(per_item):
    """More items than the grid's third index counts: rotary_qk has no use for it."""
    ovc = _ovc()
    q, k, _ = inputs((70001, 3, 1, 128), (70001, 3, 2, 128), 23, torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(4)
    positions = torch.randint(0, 3000, (70001, 3, 1) if per_item else (3, 1), generator=g, device=DEV)
    for x, y in zip((q, k), ovc.rotary_qk(q, k, ovc.rotary_plan(positions, axes=(128,)))):
        close(y, *formula(x, positions, (128,)))


def test_preparation_of_more_heads_than_a_grid_counts():
    ovc = _ovc()
    q, k, _ = inputs((1, 40000, 128), (1, 40000, 128), 24, torch.bfloat16)
    plan = ovc.rotary_plan(torch.full((1, 1), 7, device=DEV), axes=(128,))
    got, few = ovc.prepare_fp8(q, k, k, rotary=plan), ovc.prepare_fp8(q[:, -3:], k[:, -3:], k[:, -3:], rotary=plan)
    for a, b in zip((got.q, got.k, got.v), (few.q, few.k, few.v)):
        assert torch.equal(a[:, -3:].view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(got.q_descale[:, -3:], few.q_descale) and torch.equal(got.k_descale[:, -3:], few.k_descale)


@pytest.mark.parametrize("batch,s,h", [(1, 300, 2), (3, 129, 2), (2, 500, 3)])
@pytest.mark.parametrize("kind", ["int32", "int64", "float32"])
@pytest.mark.parametrize("per_item", [False, True])
@pytest.mark.parametrize("interleaved,axes,norm", [(True, (44, 42, 42), True), (False, (128,), False)])
def test_preparation_takes_every_kind_of_positions(batch, s, h, kind, per_item, interleaved, axes, norm):
    """Tolerances as in test_preparation_rotates_what_it_quantises."""
    ovc = _ovc()
    q, k, (qw, kw) = inputs((batch, s, h, 128), (batch, s, h, 128), 31 + s, torch.bfloat16)
    positions = torch.randint(-3000, 200000, (batch, s, len(axes)) if per_item else (s, len(axes)), device=DEV,
                              generator=torch.Generator(device=DEV).manual_seed(6))
    positions = positions.float() / 7.0 if kind == "float32" else positions.to(getattr(torch, kind))
    plan = ovc.rotary_plan(positions, axes=axes, interleaved=interleaved, q_weight=qw if norm else None, k_weight=kw if norm else None)
    got = ovc.prepare_fp8(q, k, k, rotary=plan)
    blocks = -(-s // 128)
    for x, w, codes, descale in ((q, qw, got.q, got.q_descale), (k, kw, got.k, got.k_descale)):
        want, size = formula(x, positions, axes, interleaved, weight=w if norm else None)
        longest, top = [torch.nn.functional.pad(t, (0, 0, 0, 0, 0, blocks * 128 - s)).view(batch, blocks, 128, h, 128).amax((2, 4)).transpose(1, 2)
                        for t in (size, want.abs())]
        d = descale.double()
        assert bool(((d * 448 - top).abs() <= F32 * longest + 4 * 2.0 ** -24 * top).all())
        per_token = d.transpose(1, 2).repeat_interleave(128, 1)[:, :s, :, None]
        value, off = want / per_token, F32 * size / per_token + 4 * 2.0 ** -24 * (want / per_token).abs()
        limit = (value.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) + 1.1 * off
        assert bool(((codes.double().view(batch, s, h, 128) - value).abs() <= limit).all())
    if not per_item and batch > 1:  # an item by itself
        one = ovc.prepare_fp8(q[1], k[1], k[1], rotary=plan)
        assert torch.equal(one.q.view(torch.uint8), got.q[1].view(torch.uint8)) and torch.equal(one.k_descale[0], got.k_descale[1])
