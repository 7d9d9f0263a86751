"""Front ends on the host: which stream a call's workspace is cleared on."""
import pytest
import torch

from apertura_amd import decode, prefix, scored
from apertura_amd.decode import DecodeStep
from apertura_amd.prefix import PrefixStep
from apertura_amd.scored import Score

BF = torch.bfloat16


class _Found(Exception):
    pass


@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("call", ["decode_step", "decode_raw", "decode_raw_q8", "scored_decode", "prefix_decode"])
def test_a_new_workspace_is_cleared_on_the_launch_s_stream(monkeypatch, call, given):
    """torch.zeros on another stream than the launch's could clear partials that the launch has written:
    the fill is ordered with it, on its stream."""
    current = []

    class Entered:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            current.append(self.stream)

        def __exit__(self, *_):
            current.pop()

    def workspace(*_):
        raise _Found(current[-1] if current else None)

    monkeypatch.setattr(torch.cuda, "stream", Entered)
    for module, name in ((decode, "new_workspace"), (decode, "new_raw_workspace"), (scored, "new_workspace"),
                         (prefix, "new_prefix_workspace")):
        monkeypatch.setattr(module, name, workspace)
    monkeypatch.setattr(decode, "_check_cache", lambda *a: None)
    B, hq, hkv, D, cap = 2, 4, 2, 512, 32
    q, new, pos = torch.zeros(B, hq, D, dtype=BF), torch.zeros(B, hkv, D, dtype=BF), torch.zeros(B, dtype=torch.int32)
    cache, step = torch.zeros(B, hkv, cap, D, dtype=BF), DecodeStep(B, hq, hkv, D, cap)
    kw, inv = torch.zeros(D, dtype=BF), torch.zeros(256)
    side = object() if given else None
    calls = {
        "decode_step": lambda: decode.decode_step(step, q, new, new, cache, cache.clone(), pos, stream=side),
        "decode_raw": lambda: decode.decode_raw(decode.RawStep(B, hq, hkv, cap), q, new, cache, pos, kw, inv, stream=side),
        "decode_raw_q8": lambda: decode.decode_raw_q8(
            decode.RawStep(B, hq, hkv, cap), q, new, torch.zeros(B, hkv, cap, D, dtype=torch.uint8),
            torch.zeros(B, hkv, cap), torch.zeros(B, hkv, cap), pos, kw, inv, stream=side),
        "scored_decode": lambda: scored.scored_decode(step, Score(), q, new, new, cache, cache.clone(), pos, stream=side),
        "prefix_decode": lambda: prefix.prefix_decode(PrefixStep(step, 8), q, new, new, torch.zeros(hkv, 8, D, dtype=BF),
                                                      torch.zeros(hkv, 8, D, dtype=BF), cache, cache.clone(), pos, stream=side),
    }
    with pytest.raises(_Found) as at:
        calls[call]()
    assert at.value.args[0] is side


@pytest.mark.gpu
def test_calls_on_a_stream_beside_a_busy_one():
    """One-shot calls on a side stream, their workspaces their own, while the current stream is asleep:
    done when the side stream is, and as on the current one."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    rows = lambda *shape: torch.randn(shape, device="cuda", generator=g).to(BF)
    B, hq, hkv, D, cap = 3, 8, 2, 128, 400
    step = DecodeStep(B, hq, hkv, D, cap, scale=D ** -0.5)
    q, kn, vn, kc, vc = rows(B, hq, D), rows(B, hkv, D), rows(B, hkv, D), rows(B, hkv, cap, D), rows(B, hkv, cap, D)
    pk, pv = rows(hkv, 300, D), rows(hkv, 300, D)
    pos = torch.tensor([399, 7, 200], dtype=torch.int32, device="cuda")
    pstep, ppos = PrefixStep.for_caches(pk, kc, hq, scale=D ** -0.5), pos + 300
    calls = [lambda s: decode.decode_step(step, q, kn, vn, kc, vc, pos, stream=s),
             lambda s: scored.scored_decode(step, Score(20.0), q, kn, vn, kc, vc, pos, stream=s),
             lambda s: prefix.prefix_decode(pstep, q, kn, vn, pk, pv, kc, vc, ppos, stream=s)]
    want = [f(None) for f in calls]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for f, w in zip(calls, want):
        torch.cuda._sleep(20_000_000)
        got = [f(side) for _ in range(5)]
        side.synchronize()
        with torch.cuda.stream(side):
            assert all(torch.equal(x, w) for x in got)
        torch.cuda.synchronize()
        assert all(torch.equal(x, w) for x in got)
