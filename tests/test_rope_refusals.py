"""What the append-with-rotation entry points refuse, before any device work."""

import numpy as np
import pytest
import torch

from easydel_amd import _lib, kernels

A = 0x7000_0000_0000


def _call(lib, **over):
    v = dict(q=A, k=A, v=A, out=A + 64, pages=A, scales=None, table=A, pos=None, ctx=A, bt=A, qsl=A, ns=A, T=4, S=2, M=8, P=16, pg=64, Hq=8, Hkv=2, D=64,
             Dp=64, C=4, rope=64, rows=100, neox=1, qs=512, ks=128, vs=128, src=1, kv=1)
    v.update(over)
    return lib.rpa_rope_page_scatter_ragged(None, v["q"], v["k"], v["v"], v["out"], v["pages"], v["scales"], v["table"], v["pos"], v["ctx"], v["bt"], v["qsl"],
                                            v["ns"], v["T"], v["S"], v["M"], v["P"], v["pg"], v["Hq"], v["Hkv"], v["D"], v["Dp"], v["C"], v["rope"], v["rows"],
                                            v["neox"], v["qs"], v["ks"], v["vs"], v["src"], v["kv"])


BAD = [(dict(rope=63), "rope_dim", -1), (dict(rope=66), "rope_dim", -1), (dict(rope=0), "bad size", -1), (dict(rows=0), "table_rows=0", -1), (dict(neox=2), "neox", -1),
       (dict(src=2), "source dtype", -2), (dict(kv=5), "page dtype", -2), (dict(kv=3), "int8 KV pages need kv_scales", -1), (dict(scales=A), "not 8-bit", -1),
       (dict(C=3), "combined heads", -1), (dict(Dp=32), "Dp=32", -1), (dict(qs=511), "overlap", -1), (dict(ks=127), "overlap", -1), (dict(vs=0), "overlap", -1),
       (dict(q=None), "null", -1), (dict(v=None), "null", -1), (dict(ns=None), "null", -1), (dict(table=None), "null", -1), (dict(q=A + 1), "aligned", -1),
       (dict(table=A + 2), "aligned", -1), (dict(pages=A + 2), "4 bytes", -1), (dict(out=A, qs=600), "not contiguous", -1),
       (dict(M=1 << 26), "2^31", -2), (dict(S=1 << 30), "too many", -2), (dict(T=-1), "bad size", -1), (dict(Hq=0), "bad size", -1)]


@pytest.mark.parametrize("over,text,code", BAD)
def test_the_c_entry_refuses(over, text, code):
    lib = _lib.load()
    assert _call(lib, **over) == code
    assert text in lib.rpa_last_error().decode()


def test_an_empty_batch_is_a_no_op():
    assert _call(_lib.load(), T=0) == 0


def test_pools_and_latent_pages_refuse():
    lib = _lib.load()
    base = [None, A, A, A, A + 64, A, A, A, None, A, A, A, None, 4, 2, 8, 16, 64, 8, 2, 64, 64, 100, 1, 512, 128, 128, 1]
    assert lib.rpa_rope_unified_page_scatter(*base, 3) == _lib.RPA_ERR_UNSUPPORTED and b"int8" in lib.rpa_last_error()
    bad = list(base)
    bad[6] = None
    assert lib.rpa_rope_unified_page_scatter(*bad, 1) == _lib.RPA_ERR_INVALID_ARGUMENT
    latent = [None, A, A, A, A + 64, A, A, None, A, A, A, A, 4, 2, 8, 16, 64, 8, 512, 64, 640, 100, 1, 512, 64, 1]
    bad = list(latent)
    bad[20] = 600 - 32
    assert lib.rpa_rope_mla_page_scatter(*bad, 1) == _lib.RPA_ERR_INVALID_ARGUMENT and b"row_elems" in lib.rpa_last_error()
    bad = list(latent)
    bad[20] = 642
    assert lib.rpa_rope_mla_page_scatter(*bad, 1) == _lib.RPA_ERR_UNSUPPORTED and b"multiple of 4" in lib.rpa_last_error()
    assert lib.rpa_rope_mla_page_scatter(*latent, 3) == _lib.RPA_ERR_UNSUPPORTED
    bad = list(latent)
    bad[19] = 0
    assert lib.rpa_rope_mla_page_scatter(*bad, 1) == _lib.RPA_ERR_INVALID_ARGUMENT


def test_tensors_off_the_gpu_and_wrong_shapes_are_refused():
    q, k = torch.zeros(4, 8, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    pages, tab = torch.zeros(8, 16, 4, 64, dtype=torch.bfloat16), torch.zeros(10, 64)
    i = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    call = lambda q=q, k=k, v=k, pages=pages, tab=tab, **kw: kernels.rope_page_scatter_ragged(q, k, v, pages, tab, i(4), i(0), i(0, 4), i(1), **kw)  # noqa: E731
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()
    with pytest.raises(ValueError, match="expected"):
        call(v=k[:, :1])
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        call(q=q.double())


def test_overlap_and_stride_checks_of_the_wrapper():
    """The host arithmetic behind the checks, on CPU tensors."""
    buf = torch.zeros(4, 10, 64)
    assert kernels._span(buf) == (buf.data_ptr(), buf.data_ptr() + 4 * 10 * 64 * 4)
    view = buf[:, 2:4]
    assert kernels._span(view) == (buf.data_ptr() + 2 * 64 * 4, buf.data_ptr() + (3 * 640 + 3 * 64 + 64) * 4)
    with pytest.raises(ValueError, match="overlaps"):
        kernels._turned_out(buf[:, :2], buf.reshape(-1)[64:64 + 512].reshape(4, 2, 64), (), "query_out")
    whole = torch.zeros(4, 2, 64)
    assert kernels._turned_out(whole, whole, (), "query_out") is whole
    with pytest.raises(ValueError, match="overlaps"):
        kernels._turned_out(whole, whole, (whole[:1],), "query_out")
    with pytest.raises(ValueError, match="contiguous"):
        kernels._turned_out(whole, torch.zeros(4, 64, 2).transpose(1, 2), (), "query_out")
    with pytest.raises(ValueError, match="rope_dim"):
        kernels._table(torch.zeros(4, 3), None, 64, whole.device)
    with pytest.raises(ValueError, match="rope part"):
        kernels._table(torch.zeros(4, 32), 64, 64, whole.device)


def test_the_rotation_oracle_turns_by_the_angle():
    from rope_testlib import rotate, table

    tab = table(50, 8)
    x = np.random.default_rng(0).standard_normal((50, 1, 8))
    for neox in (True, False):
        y = rotate(x, tab, 8, neox, np.float64)
        pair = (lambda a: a[..., :4] + 1j * a[..., 4:]) if neox else (lambda a: a[..., 0::2] + 1j * a[..., 1::2])
        angle = np.arange(50)[:, None, None] * 10000.0 ** (-np.arange(0, 8, 2) / 8)
        assert np.abs(pair(y) - pair(x) * np.exp(1j * angle)).max() < 1e-6


def _unchecked(monkeypatch):
    """The wrappers on CPU tensors: everything but where memory lies."""
    def rows(t, name, shape, dtype, device):
        return t.data_ptr(), t.stride(0)

    monkeypatch.setattr(kernels, "_rows", rows)
    monkeypatch.setattr(kernels, "_on", lambda t, *a: t.data_ptr())
    monkeypatch.setattr(kernels, "_launch", lambda *a: None)


I = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731


@pytest.mark.parametrize("what", ["pages", "scales", "table", "positions", "context_lens", "pool", "latent"])
def test_turned_queries_may_not_go_into_any_operand(monkeypatch, what):
    """``query_out`` inside the pages, the scales, the table or the metadata."""
    _unchecked(monkeypatch)
    q, k = torch.zeros(2, 2, 64), torch.zeros(2, 1, 64)
    inside = torch.zeros(4096)
    out = inside[256:512].view(2, 2, 64)
    pages, table = torch.zeros(2, 4, 2, 64), torch.zeros(10, 64)
    meta = dict(context_lens=I(2), block_tables=I(0), query_start_loc=I(0, 2), num_seqs=I(1))
    with pytest.raises(ValueError, match="query_out overlaps another operand"):
        if what == "pages":
            kernels.rope_page_scatter_ragged(q, k, k, inside[:1024].view(2, 4, 2, 64), table, **meta, query_out=out)
        elif what == "scales":
            kernels.rope_page_scatter_ragged(q, k, k, torch.zeros(256, 4, 2, 64, dtype=torch.int8), table, **meta, kv_scales=inside[:512], query_out=out)
        elif what == "table":
            kernels.rope_page_scatter_ragged(q, k, k, pages, inside[:640].view(10, 64), **meta, query_out=out)
        elif what == "positions":
            kernels.rope_page_scatter_ragged(q, k, k, pages, table, **meta, positions=inside.view(torch.int32)[300:302], query_out=out)
        elif what == "context_lens":
            kernels.rope_page_scatter_ragged(q, k, k, pages, table, **{**meta, "context_lens": inside.view(torch.int32)[511:512]}, query_out=out)
        elif what == "pool":
            kernels.rope_unified_page_scatter(q, k, k, torch.zeros(4, 4, 1, 64), inside[:1024].view(4, 4, 1, 64), table, **meta, query_out=out)
        else:
            kernels.rope_mla_page_scatter(q, torch.zeros(2, 128), k[:, 0], inside[:1024].view(1, 4, 256), table, **meta, query_out=out)
    for fine in (None, q, inside[1024:1280].view(2, 2, 64)):  # beside them is fine
        got, _ = kernels.rope_page_scatter_ragged(q, k, k, inside[:1024].view(2, 4, 2, 64), table, **meta, query_out=fine)
        assert fine is None or got is fine
    with pytest.raises(ValueError, match="overlaps another operand"):  # in place, too
        kernels.rope_page_scatter_ragged(out, k, k, inside[:1024].view(2, 4, 2, 64), table, **meta, query_out=out)
