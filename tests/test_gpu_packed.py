"""attention_packed against the definition in 64 bits.

Tolerances, per element.  u = half a step of the type (2^-8 bf16, 2^-11 fp16).  With p the exact probabilities and A the attention
of |V| (A = sum p |v|, so |out| <= A): rounding each probability to 16 bits moves the result by at most u A (fp16 also by
2^-25 max|v| for each probability below its normal range), rounding the result by u |out|.  A score is a float32 sum of 128
products, off by at most 130 * 2^-24 * sum |q k| scale =: d, twice that with the sum's own error; exponentials and the
sums are off by 2^-21 and (n / 8 + 64) 2^-24 relative.  All of those multiply A; together e = 2 d + 2^-20 + (n / 8 + 64) 2^-23.
lse: absolute error e, and 2^-22 of its value.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from gpu_util import DEV  # noqa: E402

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _ovc():
    import open_vc_attn

    return open_vc_attn


def _check_status():
    from open_vc_attn.forward import check_status

    check_status(torch.device(DEV))


def cumulative(lens, device=DEV):
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=device)


def definition(q, k, v, q_lens, k_lens, causal, scale=None):
    """out, A, lse, score error bound d (see above), all float64; rows behind the last sequence: zero, -inf."""
    scale = 128 ** -0.5 if scale is None else scale
    g = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size, most = out.clone(), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    a = c = 0
    for lq, lk in zip(q_lens, k_lens):
        qs, ks, vs = q[a:a + lq].double(), k[c:c + lk].double(), v[c:c + lk].double()
        for h in range(q.shape[1] if lq and lk else 0):
            s = qs[:, h] @ ks[:, h // g].T * scale
            if causal:
                seen = torch.arange(lk, device=q.device)[None] < (torch.arange(lq, device=q.device) + 1 + lk - lq)[:, None]
                s = s.masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1).nan_to_num()  # rows that see nothing
            out[a:a + lq, h], size[a:a + lq, h] = p @ vs[:, h // g], p @ vs[:, h // g].abs()
            lse[a:a + lq, h] = torch.logsumexp(s, -1)
            most[a:a + lq, h] = (qs[:, h].abs() @ ks[:, h // g].abs().T).amax(-1) * abs(scale)
        a, c = a + lq, c + lk
    return out, size, lse.t(), 130 * 2.0 ** -24 * most


def close(out, lse, q, k, v, q_lens, k_lens, causal, scale=None):
    want, size, want_lse, d = definition(q, k, v, q_lens, k_lens, causal, scale)
    n = max(k_lens)
    e = 2 * d + 2.0 ** -20 + (n / 8 + 64) * 2.0 ** -23
    u = U[q.dtype]
    limit = (u + e[..., None]) * size * (1 + u) + u * want.abs() + e[..., None] * want.abs()
    if q.dtype == torch.float16:
        limit = limit + n * 2.0 ** -25 * v.double().abs().max() + 2.0 ** -25
    off = (out.double() - want).abs()
    assert bool((off <= limit).all()), float((off - limit).max())
    if lse is not None:
        empty = want_lse == -math.inf
        assert torch.equal(empty, lse == -math.inf)
        off = (lse.double() - want_lse).abs()[~empty]
        assert bool((off <= (e.t() + 2.0 ** -22 * want_lse.abs())[~empty]).all())


def inputs(q_lens, k_lens, hq, hk, dtype, seed, extra=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(sum(q_lens) + extra, hq, 128, generator=g, device=DEV).to(dtype)
    k, v = [torch.randn(sum(k_lens) + extra, hk, 128, generator=g, device=DEV).to(dtype) for _ in range(2)]
    return q, k, v


LENGTHS = [
    ([1], [1]), ([1], [128]), ([1], [129]), ([127], [127]), ([128], [128]), ([129], [129]), ([257], [257]), ([300], [5]),
    ([5], [300]), ([500, 3, 0, 77], [500, 3, 0, 77]), ([40, 3, 9, 200], [0, 700, 8, 1]), ([1] * 5, [1, 2000, 129, 0, 640]),
    ([2, 1, 4], [3000, 1, 1111]), ([60, 300], [3000, 1500]), ([700, 900], [700, 900]), ([1] * 40, [3] * 40),
]


@pytest.mark.parametrize("q_lens,k_lens", LENGTHS)
@pytest.mark.parametrize("hq,hk,dtype", [(1, 1, torch.bfloat16), (8, 2, torch.bfloat16), (9, 3, torch.float16), (7, 1, torch.float16),
                                         (24, 24, torch.bfloat16)])
@pytest.mark.parametrize("causal", [False, True])
def test_matches_the_definition(q_lens, k_lens, hq, hk, dtype, causal):
    ovc = _ovc()
    q, k, v = inputs(q_lens, k_lens, hq, hk, dtype, sum(q_lens) + hq)
    cu = cumulative(q_lens), cumulative(k_lens)
    out, lse = ovc.attention_packed(q, k, v, *cu, causal=causal, return_lse=True)
    _check_status()
    assert out.dtype == dtype and out.shape == q.shape and lse.shape == (hq, q.shape[0]) and lse.dtype == torch.float32
    close(out, lse, q, k, v, q_lens, k_lens, causal)
    assert torch.equal(out, ovc.attention_packed(q, k, v, *cu, causal=causal))


@pytest.mark.parametrize("hq,hk", [(5, 1), (48, 1), (128, 1), (130, 2), (64, 1), (65, 1)])
@pytest.mark.parametrize("q_lens,k_lens", [([3, 70], [400, 90]), ([150], [150])])
def test_group_sizes(hq, hk, q_lens, k_lens):
    ovc = _ovc()
    q, k, v = inputs(q_lens, k_lens, hq, hk, torch.bfloat16, hq)
    out, lse = ovc.attention_packed(q, k, v, cumulative(q_lens), cumulative(k_lens), causal=True, return_lse=True)
    _check_status()
    close(out, lse, q, k, v, q_lens, k_lens, True)


@pytest.mark.parametrize("scale", [1e-3, 0.5, 3.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_and_peaked_rows(scale, dtype):
    """Large scales make single keys win, and move the running maximum by more than the 2^8 that it may lag behind."""
    ovc = _ovc()
    lens = [900, 33]
    q, k, v = inputs(lens, lens, 4, 2, dtype, 11)
    k = (k.float() * torch.linspace(0.1, 3.0, k.shape[0], device=DEV)[:, None, None]).to(dtype)
    out, lse = ovc.attention_packed(q, k, v, cumulative(lens), softmax_scale=scale, return_lse=True)
    _check_status()
    close(out, lse, q, k, v, lens, lens, False, scale)


@pytest.mark.parametrize("lens", [[200, 77, 300], [1, 1, 1]])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_other_sequences_and_padding_never_reach_a_row(lens, bad):
    """The middle sequence and the rows behind the last one hold values that are not finite."""
    ovc = _ovc()
    k_lens = [n * 7 for n in lens]
    q, k, v = inputs(lens, k_lens, 4, 2, torch.bfloat16, 5, extra=50)
    cu = cumulative(lens), cumulative(k_lens)
    clean = ovc.attention_packed(q, k, v, *cu, causal=True)
    a, b, c, d = lens[0], lens[0] + lens[1], k_lens[0], k_lens[0] + k_lens[1]
    for t, lo, hi, end in ((q, a, b, sum(lens)), (k, c, d, sum(k_lens)), (v, c, d, sum(k_lens))):
        t[lo:hi] = bad
        t[end:] = bad
    out, lse = ovc.attention_packed(q, k, v, *cu, causal=True, return_lse=True)
    _check_status()
    assert torch.equal(out[:a], clean[:a]) and torch.equal(out[b:sum(lens)], clean[b:sum(lens)])
    assert bool(out[a:b].isnan().all()) and not out[sum(lens):].any() and bool((lse[:, sum(lens):] == -math.inf).all())


@pytest.mark.parametrize("q_lens,k_lens", [([300, 40], [300, 40]), ([1, 2], [4000, 300])])
def test_rows_behind_the_last_sequence(q_lens, k_lens):
    ovc = _ovc()
    q, k, v = inputs(q_lens, k_lens, 4, 1, torch.float16, 6, extra=700)
    cu = cumulative(q_lens), cumulative(k_lens)
    fresh = ovc.attention_packed(q, k, v, *cu)
    end = sum(q_lens)
    assert not fresh[end:].any()
    out = torch.full_like(q, 7.0)
    assert ovc.attention_packed(q, k, v, *cu, out=out) is out
    _check_status()
    assert torch.equal(out[:end], fresh[:end]) and bool((out[end:] == 7.0).all())
    for tensors in ((q, k[:0], v[:0]), (q[:0], k, v)):  # no keys at all; no rows at all
        none, lse = ovc.attention_packed(*tensors, *cu, return_lse=True)
        assert not none.any() and bool((lse == -math.inf).all())
    assert bool((ovc.attention_packed(q, k[:0], v[:0], *cu, out=out)[end:] == 7.0).all()) and not out[:end].any()


def test_bounds_that_lie_stay_inside_the_tensors():
    """Every bound is clamped to its tensor before it is used (the kernels' bounds()): wrong rows, nothing worse.  (All rows may
    be wrong: where the rows end, and how the keys are split, comes of all bounds together.)"""
    ovc = _ovc()
    q, k, v = inputs([300], [3000], 4, 2, torch.bfloat16, 8)
    good = ovc.attention_packed(q, k, v, cumulative([100, 200]), cumulative([1000, 2000]))
    for bounds in ([0, 100, 2 ** 31 - 1], [0, 100, -5], [0, -2 ** 31, 300], [0, 300, 0, 300, 0, 300, 0, 300, 0, 300]):
        cq = torch.tensor(bounds, dtype=torch.int32, device=DEV)
        ck = torch.tensor([min(10 * x, 2 ** 31 - 1) if x > 0 else x for x in bounds], dtype=torch.int32, device=DEV)
        out, lse = ovc.attention_packed(q, k, v, cq, ck, causal=True, return_lse=True)
        _check_status()
        assert out.shape == q.shape
        assert ovc.attention_packed(q, k, v, cq, ck, out=out) is out
        _check_status()
    assert torch.equal(good, ovc.attention_packed(q, k, v, cumulative([100, 200]), cumulative([1000, 2000])))


@pytest.mark.parametrize("causal", [False, True])
def test_slices_strides_and_shared_storage(causal):
    ovc = _ovc()
    g = torch.Generator(device=DEV).manual_seed(21)
    lens = [210, 99]
    cu = cumulative(lens)
    qkv = torch.randn(309, 12, 128, generator=g, device=DEV).to(torch.bfloat16)
    q, k, v = qkv.split([8, 2, 2], 1)
    want = ovc.attention_packed(q.contiguous(), k.contiguous(), v.contiguous(), cu, causal=causal)
    assert torch.equal(ovc.attention_packed(q, k, v, cu, causal=causal), want)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(ovc.attention_packed(*heads_first, cu, causal=causal), want)
    shared = k[:, :1].expand(309, 2, 128)  # stride 0: copied
    assert torch.equal(ovc.attention_packed(q, shared, v, cu, causal=causal),
                       ovc.attention_packed(q, shared.contiguous(), v, cu, causal=causal))
    odd = torch.randn(309, 12, 132, generator=g, device=DEV).to(torch.bfloat16)[..., 2:130].split([8, 2, 2], 1)  # off the 16-byte grid
    assert torch.equal(ovc.attention_packed(*odd, cu, causal=causal), ovc.attention_packed(*[t.contiguous() for t in odd], cu, causal=causal))
    single = qkv[:1, :8], qkv[:1, 8:9], qkv[:1, 9:10]  # one token, one key head: strides of size-1 dimensions mean nothing
    assert torch.equal(ovc.attention_packed(*single, cumulative([1])), qkv[:1, 9:10].expand(1, 8, 128))
    same = ovc.attention_packed(k, k, k, cu, causal=causal)
    assert torch.equal(same, ovc.attention_packed(k.clone(), k.clone(), k.clone(), cu, causal=causal))


@pytest.mark.parametrize("q_lens,k_lens", [([400, 30], [400, 30]), ([1, 1, 1], [5000, 70, 900])])
def test_captured_replayed_and_on_other_streams(q_lens, k_lens):
    """A replay reads lengths and values anew; two graphs and two streams do not share a workspace."""
    ovc = _ovc()
    q, k, v = inputs(q_lens, k_lens, 8, 2, torch.bfloat16, 9)
    cu_q, cu_k = cumulative(q_lens), cumulative(k_lens)
    call = lambda: ovc.attention_packed(q, k, v, cu_q, cu_k, causal=True, return_lse=True)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [call() for _ in range(3)]
    here = [call() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for got in other + here for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for change in (False, True):
        if change:
            k_lens = [max(0, n - 60) for n in k_lens]
            cu_k.copy_(cumulative(k_lens))
            q.copy_(torch.randn_like(q.float()).to(q.dtype))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        _check_status()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, call()))
            close(out[0], out[1], q, k, v, q_lens, k_lens, True)


def test_prompt_then_tokens_with_rotary_positions():
    """The operators as a model uses them: slices of a projection are normalised and rotated, a packed prompt is attended, then
    one token of each request at a time behind its keys; the tokens' rows equal the prompt's within both calls' roundings."""
    ovc = _ovc()
    g = torch.Generator(device=DEV).manual_seed(31)
    lens, hq, hk = [700, 5, 260], 8, 2
    total = sum(lens)
    q, k, v = torch.randn(total, hq + 2 * hk, 128, generator=g, device=DEV).to(torch.bfloat16).split([hq, hk, hk], 1)
    at = torch.cat([torch.arange(n, device=DEV) for n in lens])[:, None]
    weight = 1 + 0.1 * torch.randn(128, generator=g, device=DEV)
    qr, kr = ovc.rotary_qk(q, k, ovc.rotary_plan(at, axes=(128,), interleaved=False, q_weight=weight, k_weight=weight))
    cu = cumulative(lens)
    whole, lse = ovc.attention_packed(qr, kr, v, cu, causal=True, return_lse=True)
    close(whole, lse, qr, kr, v, lens, lens, True)
    ends = (cu[1:] - 1).long()
    one = ovc.rotary_qk(q[ends], k[ends], ovc.rotary_plan(at[ends], axes=(128,), interleaved=False, q_weight=weight, k_weight=weight))
    assert torch.equal(one[0], qr[ends]) and torch.equal(one[1], kr[ends])
    step, step_lse = ovc.attention_packed(one[0], kr, v, cumulative([1] * 3), cu, causal=True, return_lse=True)
    close(step, step_lse, one[0], kr, v, [1] * 3, lens, True)
    _check_status()


def test_keys_behind_the_32_bit_range():
    """1.1e6 rows of 16 key heads of 128 values: element offsets pass 2^31."""
    ovc = _ovc()
    n, h = 1100000, 16
    k = torch.zeros(n, h, 128, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    tail = 1000
    g = torch.Generator(device=DEV).manual_seed(2)
    k[-tail:] = torch.randn(tail, h, 128, generator=g, device=DEV).to(k.dtype)
    v[-tail:] = torch.randn(tail, h, 128, generator=g, device=DEV).to(k.dtype)
    q = torch.randn(2, h, 128, generator=g, device=DEV).to(k.dtype)
    out, lse = ovc.attention_packed(q, k, v, cumulative([1, 1]), cumulative([n - tail, tail]), return_lse=True)
    _check_status()
    close(out[1:], lse[:, 1:], q[1:], k[-tail:], v[-tail:], [1], [tail], False)
    assert not out[0].any() and torch.allclose(lse[:, 0], torch.tensor(math.log(n - tail), device=DEV), rtol=2.0 ** -15)


def test_refusals():
    ovc = _ovc()
    q, k, v = inputs([8], [8], 4, 2, torch.bfloat16, 1)
    cu = cumulative([8])
    cases = [
        ((q[0], k, v, cu), {}, "packed"), ((q[..., :64], k, v, cu), {}, "packed"), ((q, k, v[:4], cu), {}, "match"),
        ((q[:, :3], k, v, cu), {}, "multiple"), ((q[:, :1], k, v, cu), {}, "multiple"), ((q, k.half(), v.half(), cu), {}, "matching"),
        ((q.float(), k.float(), v.float(), cu), {}, "matching"), ((q, k, v, cu.long()), {}, "cu_seqlens_q"),
        ((q, k, v, cu[:1]), {}, "cu_seqlens_q"), ((q, k, v, cu.cpu()), {}, "reside"), ((q, k, v, [0, 8]), {}, "cu_seqlens_q"),
        ((q, k, v, cu, cumulative([4, 4])), {}, "same number"), ((q, k, v, cu), dict(softmax_scale=0.0), "softmax_scale"),
        ((q, k, v, cu), dict(softmax_scale=math.nan), "softmax_scale"), ((q, k, v, cu), dict(out=q.float()), "out must"),
        ((q, k, v, cu), dict(out=q.transpose(0, 1).contiguous().transpose(0, 1)), "out must"), ((q.cpu(), k, v, cu), {}, "same CUDA"),
        ((q.clone().requires_grad_(), k, v, cu), {}, "detach"),
    ]
    for arguments, options, match in cases:
        with pytest.raises(ValueError, match=match):
            ovc.attention_packed(*arguments, **options)


@pytest.mark.parametrize("lengths", ["rows and keys", "one token each"])
def test_many_sequences(lengths):
    """Hundreds of sequences, some empty: more than a warp looks through at a time, and more than a split launch plans for."""
    ovc = _ovc()
    g = torch.Generator().manual_seed(7)
    k_lens = torch.randint(0, 300, (333,), generator=g).tolist()
    q_lens = [1] * 333 if lengths == "one token each" else torch.randint(0, 40, (333,), generator=g).tolist()
    for count in (333, 150, 129):
        ql, kl = q_lens[:count], k_lens[:count]
        q, k, v = inputs(ql, kl, 4, 2, torch.bfloat16, count)
        out, lse = ovc.attention_packed(q, k, v, cumulative(ql), cumulative(kl), causal=True, return_lse=True)
        _check_status()
        close(out, lse, q, k, v, ql, kl, True)


@pytest.mark.parametrize("count,hk,low,high", [(40, 8, 1, 3000), (100, 2, 300, 900)])
def test_single_tokens_of_many_requests(count, hk, low, high):
    """More row tiles than SMs, each with few rows: shares of several segments."""
    ovc = _ovc()
    kl = torch.randint(low, high, (count,), generator=torch.Generator().manual_seed(count)).tolist()
    ql = [1 + i % 3 for i in range(count)]
    q, k, v = inputs(ql, kl, 4 * hk, hk, torch.float16, count)
    out, lse = ovc.attention_packed(q, k, v, cumulative(ql), cumulative(kl), causal=True, return_lse=True)
    _check_status()
    close(out, lse, q, k, v, ql, kl, True)
    assert torch.equal(out, ovc.attention_packed(q, k, v, cumulative(ql), cumulative(kl), causal=True))


def test_refuses_an_output_that_is_no_memory_of_its_own():
    ovc = _ovc()
    q, k, v = inputs([8], [8], 4, 4, torch.bfloat16, 1)
    cu = cumulative([8])
    both = torch.empty(16, 4, 128, device=q.device, dtype=q.dtype)
    fused = torch.empty(8, 3, 4, 128, device=q.device, dtype=q.dtype)
    for out, arguments in ((q, (q, k, v)), (k, (q, k, v)), (v, (q, k, v)), (both[4:12], (q, both[:8], v)), (both[4:12], (q, k, both[8:])),
                           (fused.view(24, 4, 128)[9:17], fused.unbind(1))):
        with pytest.raises(ValueError, match="share memory"):
            ovc.attention_packed(*arguments, cu, out=out)
    with pytest.raises(ValueError, match="detach"):
        ovc.attention_packed(q, k, v, cu, out=torch.empty_like(q).requires_grad_())
    both[:8] = q  # neighbours in one allocation are no overlap
    got = ovc.attention_packed(both[:8], k, v, cu, out=both[8:])
    assert torch.equal(got, ovc.attention_packed(q, k, v, cu))


@pytest.mark.parametrize("scale", [1e-40, 3e38, 1e300])
def test_refuses_scales_that_float32_cannot_hold(scale):
    q, k, v = inputs([8], [8], 2, 2, torch.float16, 1)
    with pytest.raises(ValueError, match="softmax_scale"):
        _ovc().attention_packed(q, k, v, cumulative([8]), softmax_scale=scale)


@pytest.mark.parametrize("q_lens,k_lens", [([300, 40], [300, 40]), ([1, 2], [4000, 300]), ([0, 0], [9, 0])])
@pytest.mark.parametrize("given", [False, True])
def test_lse_behind_the_last_sequence(q_lens, k_lens, given):
    ovc = _ovc()
    q, k, v = inputs(q_lens, k_lens, 4, 1, torch.float16, 6, extra=200)
    q.new_full((4, q.shape[0]), math.nan, dtype=torch.float32)  # memory that the allocator may hand out next
    _, lse = ovc.attention_packed(q, k, v, cumulative(q_lens), cumulative(k_lens), return_lse=True, out=torch.empty_like(q) if given else None)
    end = sum(q_lens)
    assert bool((lse[:, end:] == -math.inf).all()) and bool(torch.isfinite(lse[:, :end]).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("split", [False, True])
def test_many_small_probabilities_beside_a_large_one(dtype, split):
    """One key whose probability is 2^26 times that of each of 200000 others, which hold 0.3 per cent of the row together."""
    ovc = _ovc()
    n, rows, h = 200000, 1 if split else 300, 8
    q, k = [torch.zeros(t, h, 128, device=DEV, dtype=dtype) for t in (rows, n)]
    q[..., 0], k[70000, :, 0], k[70000, :, 1] = 1.0, 18.0, 1.0
    scale = math.log(2.0) * 26 / 18
    v = torch.full_like(k, 1.0)
    v[70000] = 0.0
    out, lse = ovc.attention_packed(q, k, v, cumulative([rows]), cumulative([n]), softmax_scale=scale, return_lse=True)
    _check_status()
    small = (n - 1) * 2.0 ** -26
    want = small / (1 + small)
    # The score is exact, its product with the scale off by 2^-24 of 26 twice (scale rounded, product rounded): 2^-18 for the
    # probabilities.  fp16 steps there are 2^-24 with the factor 2^7 or none: 2^-19 / 2^-24 is whole.  Sums of n terms: n / 8
    # roundings at most in an accumulator of the tensor cores.  The sum of the row rounds once for a tile of 128 keys.
    bound = 2.0 ** -18 + (n / 8) * 2.0 ** -23 + U[dtype]
    assert bool(((out.double() - want).abs() <= bound * want).all())
    assert bool(((lse.double() - (26 * math.log(2.0) + math.log1p(small))).abs() <= 2.0 ** -18 + 19 * 2.0 ** -24 + n / 128 * 2.0 ** -24).all())


@pytest.mark.parametrize("q_lens,k_lens,hq,hk", [
    ([300], [5], 8, 2), ([200, 700], [0, 300], 7, 1),  # whole
    ([900], [600], 2, 2),  # wide split
    ([40, 40, 40], [5, 20, 700], 2, 2),  # narrow split
])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_without_keys_beside_values_that_are_not_finite(q_lens, k_lens, hq, hk, bad, dtype):
    """Every sequence's first value is not finite: a row that sees a key sees it, a row that sees none is zero all the same."""
    ovc = _ovc()
    q, k, v = inputs(q_lens, k_lens, hq, hk, dtype, 17)
    cu_q, cu_k = cumulative(q_lens), cumulative(k_lens)
    v[cu_k[:-1].long().clamp_max(v.shape[0] - 1)] = bad
    out, lse = ovc.attention_packed(q, k, v, cu_q, cu_k, causal=True, return_lse=True)
    _check_status()
    blind = torch.cat([torch.arange(a, device=DEV) + b < a for a, b in zip(q_lens, k_lens)])
    assert bool(blind.any()) and not bool(blind.all())
    assert not out[blind].any() and bool((lse[:, blind] == -math.inf).all())
    assert not bool(torch.isfinite(out[~blind]).any()) and bool(torch.isfinite(lse[:, ~blind]).all())


@pytest.mark.parametrize("q_lens,k_lens,hq,hk", [([9, 200], [700, 0], 37, 37), ([130, 200], [300, 9], 7, 1),  # whole
                                                 ([9, 250], [900, 300], 2, 2), ([3, 20], [900, 200], 7, 1)])  # wide, narrow split
def test_what_lies_behind_a_sequence_in_its_query_tile(q_lens, k_lens, hq, hk):
    """The next sequence's queries share a tile with the first one's last rows, and are not finite."""
    ovc = _ovc()
    q, k, v = inputs(q_lens, k_lens, hq, hk, torch.float16, 41)
    cu = cumulative(q_lens), cumulative(k_lens)
    end = q_lens[0]
    want, want_lse = ovc.attention_packed(q, k, v, *cu, return_lse=True)
    close(want[:end], want_lse[:, :end], q[:end], k[:k_lens[0]], v[:k_lens[0]], q_lens[:1], k_lens[:1], False)
    for bad in (math.nan, math.inf, -math.inf, 0.0):
        q[end:] = bad
        out, lse = ovc.attention_packed(q, k, v, *cu, return_lse=True)
        assert torch.equal(out[:end], want[:end]) and torch.equal(lse[:, :end], want_lse[:, :end])
    _check_status()


LYING = [[0, 100, 2 ** 31 - 1], [0, 100, -5], [0, -(2 ** 31), 300], [0, 300, 0, 300, 0, 300, 0, 300, 0, 300], [250, 20, 290, 7],
         [2 ** 31 - 1, -(2 ** 31), 2 ** 31 - 1], [-7, 3, 3, 299, 301, 300]]


@pytest.mark.parametrize("tq,tk,hq,hk", [(300, 300, 80, 80), (300, 200, 7, 1),  # whole
                                         (300, 3000, 4, 2), (300, 3000, 3, 3),  # wide split
                                         (30, 6000, 4, 1), (18, 3000, 9, 9)])  # narrow split
@pytest.mark.parametrize("causal", [False, True])
def test_bounds_that_lie_write_nothing_beside_the_outputs(tq, tk, hq, hk, causal):
    """Through the C entry: output, log-sum-exp and workspace are pieces of larger tensors whose other elements keep their
    values.  (That no access leaves them is shown by the clamps of bounds() and of the plan; this finds a mistake in them.)"""
    from ctypes import c_int64

    from open_vc_attn import _lib
    from open_vc_attn.forward import _status

    lib = _lib.load()
    q, k, v = inputs([tq], [tk], hq, hk, torch.bfloat16, 8)
    words, mirror = _status(torch.device(DEV))
    strides = [(c_int64 * 2)(h * 128, 128) for h in (hq, hk)]
    pad = 1024  # rows, elements
    for shape in LYING:
        cu = [torch.tensor([max(-(2 ** 31), min(2 ** 31 - 1, x * n // 300)) for x in shape], dtype=torch.int32, device=DEV) for n in (tq, tk)]
        sizes = (len(shape) - 1, tq, tk, hq, hk)
        out = torch.full((pad + tq + pad, hq, 128), 7.0, device=DEV, dtype=q.dtype)
        lse = torch.full((pad + hq * tq + pad,), 7.0, device=DEV)
        size = lib.ovc_attention_packed_workspace(*sizes)
        assert size % 4 == 0
        work = torch.full((pad + size // 4 + pad,), 7.0, device=DEV)
        for flags in (0, _lib.OVC_ATTN_ZERO_TAIL):
            _lib.check(
                lib.ovc_attention_packed(
                    q.data_ptr(), strides[0], k.data_ptr(), strides[1], v.data_ptr(), strides[1], _lib.OVC_BF16, cu[0].data_ptr(), cu[1].data_ptr(),
                    *sizes, flags | (_lib.OVC_ATTN_CAUSAL if causal else 0), 0.1, out[pad:].data_ptr(), lse[pad:].data_ptr(), work[pad:].data_ptr(),
                    words.data_ptr() + 4, mirror.data_ptr(), torch.cuda.current_stream().cuda_stream,
                ),
                "ovc_attention_packed",
            )
        _check_status()
        for t, n in ((out, tq), (lse, hq * tq), (work, size // 4)):
            assert bool((t[:pad] == 7.0).all()) and bool((t[pad + n:] == 7.0).all())
