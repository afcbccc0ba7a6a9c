"""The bounded-wait failure path, exercised without hanging or faulting anything: a self-test kernel whose wait
cannot complete runs into its (short) limit and reports it; the attention kernels share that wait."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from gpu_util import DEV, f32  # noqa: E402
from oracle import attention as oatt  # noqa: E402


def _mods():
    import open_vc_attn
    from open_vc_attn import _lib, forward

    return open_vc_attn, _lib, forward


def test_expired_wait_is_reported_and_the_next_calls_are_unaffected():
    ovc, _lib, forward = _mods()
    lib = _lib.load()
    device = torch.device(DEV)
    forward.check_status(device)  # start clean
    words = forward.status_word(device)
    gave_up = torch.zeros(1, dtype=torch.int32, device=DEV)
    with torch.cuda.device(device):
        _lib.check(lib.ovc_selftest_wait(words.data_ptr(), 200_000, gave_up.data_ptr(), _lib.stream_pointer(device)),
                   "ovc_selftest_wait")
    torch.cuda.synchronize()
    assert int(gave_up.item()) == 64  # every thread of the CTA ran into the limit and returned
    assert words.tolist() == [_lib.STATUS_WAIT_EXPIRED, _lib.STATUS_WAIT_EXPIRED]
    with pytest.raises(RuntimeError, match="bounded wait expired"):
        forward.check_status(device)
    forward.check_status(device)  # reading it cleared the sticky word

    # The context is intact and a normal call right after is correct.  The per-launch word the self-test
    # left set does not stop it: the library clears that word before every launch.
    assert int(words[0].item()) == _lib.STATUS_WAIT_EXPIRED
    torch.manual_seed(5)
    q, k, v = [torch.randn(300, 2, 128, device=DEV, dtype=torch.bfloat16) for _ in range(3)]
    out = ovc.attention(q, k, v)
    forward.check_status(device)
    assert torch.isfinite(out.float()).all()
    assert oatt.relative_l2(f32(out), oatt.exact_attention(f32(q), f32(k), f32(v))) < 0.10


def test_a_failure_surfaces_at_the_next_public_call_without_a_sync():
    ovc, _lib, forward = _mods()
    lib = _lib.load()
    device = torch.device(DEV)
    forward.check_status(device)
    words = forward.status_word(device)
    gave_up = torch.zeros(1, dtype=torch.int32, device=DEV)
    torch.manual_seed(6)
    q, k, v = [torch.randn(200, 1, 128, device=DEV, dtype=torch.bfloat16) for _ in range(3)]
    with torch.cuda.device(device):
        _lib.check(lib.ovc_selftest_wait(words.data_ptr(), 100_000, gave_up.data_ptr(), _lib.stream_pointer(device)),
                   "ovc_selftest_wait")
    first = ovc.attention(q, k, v)  # computes normally and publishes the sticky word behind it
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="bounded wait expired"):
        ovc.attention(q, k, v)  # raised from host memory, before anything is launched
    again = ovc.attention(q, k, v)
    forward.check_status(device)
    assert torch.equal(first, again)


# (q lengths, k lengths, query heads, key heads) of the forms of attention_packed: whole, wide split, narrow split
PACKED_FORMS = [([300, 40], [300, 40], 4, 2), ([300], [2000], 2, 2), ([1, 2], [4000, 300], 4, 1)]


def _packed_inputs(q_lens, k_lens, hq, hk):
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(sum(q_lens), hq, 128, generator=g, device=DEV).to(torch.bfloat16)
    k, v = [torch.randn(sum(k_lens), hk, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    cu = [torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32, device=DEV) for n in (q_lens, k_lens)]
    return q, k, v, *cu


@pytest.mark.parametrize("q_lens,k_lens,hq,hk", PACKED_FORMS)
def test_packed_launches_behind_a_failure_leave_nan_and_report_it(q_lens, k_lens, hq, hk):
    """The sticky word is set from the host, without its mirror: as a launch finds it behind one that gave up."""
    ovc, _lib, forward = _mods()
    device = torch.device(DEV)
    arguments = _packed_inputs(q_lens, k_lens, hq, hk)
    forward.check_status(device)
    want = ovc.attention_packed(*arguments, causal=True, return_lse=True)
    forward.check_status(device)
    words = forward.status_word(device)
    words[1:].fill_(_lib.STATUS_WAIT_EXPIRED)
    torch.cuda.synchronize()
    out, lse = ovc.attention_packed(*arguments, causal=True, return_lse=True)
    torch.cuda.synchronize()
    assert bool(out.isnan().all()) and bool(lse.isnan().all())
    words[1:].zero_()  # the launch itself has reported, whatever becomes of the word
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="bounded wait expired"):
        ovc.attention_packed(*arguments, causal=True)
    again = ovc.attention_packed(*arguments, causal=True, return_lse=True)
    forward.check_status(device)
    assert all(torch.equal(a, b) for a, b in zip(want, again))


@pytest.mark.parametrize("q_lens,k_lens,hq,hk", PACKED_FORMS)
@pytest.mark.parametrize("by", ["call", "check_status"])
def test_a_reported_failure_does_not_reach_another_stream(q_lens, k_lens, hq, hk, by):
    """The failure is reported on a stream that is busy; a call on another one right behind it computes."""
    ovc, _lib, forward = _mods()
    device = torch.device(DEV)
    arguments = _packed_inputs(q_lens, k_lens, hq, hk)
    forward.check_status(device)
    want = ovc.attention_packed(*arguments)
    words, mirror = forward._status(device)
    words[1:].fill_(_lib.STATUS_WAIT_EXPIRED)
    mirror.fill_(_lib.STATUS_WAIT_EXPIRED)
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        if by == "call":
            torch.cuda._sleep(20_000_000)  # about 10 ms
            with pytest.raises(RuntimeError, match="bounded wait expired"):
                ovc.attention_packed(*arguments)
        else:
            with pytest.raises(RuntimeError, match="bounded wait expired"):
                forward.check_status(device)
    with torch.cuda.stream(other):
        got = ovc.attention_packed(*arguments)
    torch.cuda.synchronize()
    assert torch.equal(want, got)
    forward.check_status(device)


def test_a_failure_found_in_a_capture_is_reported_again_behind_it():
    ovc, _lib, forward = _mods()
    device = torch.device(DEV)
    arguments = _packed_inputs(*PACKED_FORMS[0])
    forward.check_status(device)
    want = ovc.attention_packed(*arguments)
    words, mirror = forward._status(device)
    words[1:].fill_(_lib.STATUS_WAIT_EXPIRED)
    mirror.fill_(_lib.STATUS_WAIT_EXPIRED)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        arguments[0].neg()  # (so that the graph is not empty)
        with pytest.raises(RuntimeError, match="bounded wait expired"):
            ovc.attention_packed(*arguments)
    with pytest.raises(RuntimeError, match="bounded wait expired"):
        ovc.attention_packed(*arguments)
    assert torch.equal(want, ovc.attention_packed(*arguments))
    forward.check_status(device)
