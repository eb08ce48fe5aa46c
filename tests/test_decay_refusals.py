"""What the entry point of linear attention with a decay refuses, before any device work."""

import pytest
import torch

from easydel_amd import _lib, kernels

A = 0x7000_0000_0000


def _call(lib, **over):
    v = dict(q=A, k=A, v=A, g=A, state=A, si=A, so=None, ctx=None, qsl=A, ns=A, out=A, ws=None, ws_bytes=0, T=4, S=2, N=8, Hq=8, Hkv=2, Dk=64, Dv=64,
             qs=512, ks=128, vs=128, dt=1, scale=0.125)
    v.update(over)
    return lib.rpa_decay_linear_attention(None, v["q"], v["k"], v["v"], v["g"], v["state"], v["si"], v["so"], v["ctx"], v["qsl"], v["ns"], v["out"], v["ws"],
                                          v["ws_bytes"], v["T"], v["S"], v["N"], v["Hq"], v["Hkv"], v["Dk"], v["Dv"], v["qs"], v["ks"], v["vs"], v["dt"], v["scale"])


@pytest.mark.parametrize("over,text,code", [
    (dict(T=-1), "bad size", -1), (dict(S=0), "bad size", -1), (dict(N=0), "bad size", -1), (dict(Hq=7), "multiple of Hkv", -1), (dict(Dk=66), "multiples of 4", -2),
    (dict(Dv=260, vs=520), "at most 256", -2), (dict(dt=2), "dtype", -2), (dict(dt=5), "dtype", -2), (dict(scale=float("nan")), "not finite", -1),
    (dict(scale=float("inf")), "not finite", -1), (dict(qs=511), "overlap", -1), (dict(ks=0), "overlap", -1), (dict(vs=127), "overlap", -1),
    (dict(q=None), "null", -1), (dict(g=None), "null", -1), (dict(state=None), "null", -1), (dict(si=None), "null", -1), (dict(ns=None), "null", -1),
    (dict(out=A + 8), "16 bytes", -1), (dict(state=A + 4), "16 bytes", -1), (dict(k=A + 1), "aligned", -1), (dict(S=70000), "65000", -2)])
def test_the_c_entry_refuses(over, text, code):
    lib = _lib.load()
    assert _call(lib, **over) == code
    assert text in lib.rpa_last_error().decode()


def test_more_workgroups_than_a_launch_holds_are_refused():
    lib = _lib.load()
    big = dict(T=10_000_000, S=65_000, Hq=1000, Hkv=1000, Dk=4, Dv=4, qs=4000, ks=4000, vs=4000)
    assert _call(lib, **big) == -2
    assert "too many workgroups" in lib.rpa_last_error().decode()


def test_an_empty_batch_is_a_no_op():
    assert _call(_lib.load(), T=0) == 0


def test_the_wrapper_refuses():
    q, s = torch.zeros(4, 2, 64), torch.zeros(3, 2, 64, 32)
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    call = lambda q=q, k=q, v=q[..., :32], g=torch.zeros(2), s=s, **kw: kernels.decay_linear_attention(q, k, v, g, s, i(0), i(0, 4), i(1), **kw)  # noqa: E731
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()
    with pytest.raises(ValueError, match="expected"):
        call(q=q[0])
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        call(q=q.double())


@pytest.mark.parametrize("what", ["log_decay", "state_indices", "state_out_indices", "context_lens", "query_start_loc", "num_seqs"])
def test_the_output_may_not_lie_in_any_operand(monkeypatch, what):
    monkeypatch.setattr(kernels, "_rows", lambda t, *a: (t.data_ptr(), t.stride(0)))  # CPU tensors: everything but where memory lies
    monkeypatch.setattr(kernels, "_on", lambda t, *a: t.data_ptr())
    monkeypatch.setattr(kernels, "_launch", lambda *a: None)
    I = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    q, inside = torch.zeros(2, 1, 64), torch.zeros(512)
    given = dict(log_decay=torch.zeros(1), state=torch.zeros(3, 1, 64, 64), state_indices=I(0), query_start_loc=I(0, 2), num_seqs=I(1), context_lens=I(2),
                 state_out_indices=I(1))
    out = inside[128:256].view(2, 1, 64)
    got, _ = kernels.decay_linear_attention(q, q, q, **given, out=out)
    assert got is out
    given[what] = inside[254:254 + given[what].numel()].view(given[what].dtype)
    with pytest.raises(ValueError, match=f"out overlaps {what}"):
        kernels.decay_linear_attention(q, q, q, **given, out=out)
