"""GPU tests of the append-with-rotation operators: bit for bit against the rule that the header states (products and sums
rounded to float32 one by one, one rounding to the target type), and against the rotation in 64 bits."""

import numpy as np
import pytest
import torch

from easydel_amd import kernels
from rope_testlib import BF16, F16, F32, FP8, INT8, append_scaled, batch, decode, dev, encode, orc, raw_of, rotate, table, tl, token_positions

pytestmark = pytest.mark.gpu

STALE = {F32: np.float32(7.5), BF16: np.uint16(0x40F0), F16: np.float16(7.5), FP8: np.uint8(0x4F)}


def _inputs(rng, T, heads, D, tag):
    x = rng.standard_normal((T, heads, D)).astype(np.float32)
    raw = encode(x, tag)
    return raw, decode(raw, tag)


def _rows(tab, pos, positions=None):
    return tab[np.clip(pos if positions is None else positions, 0, len(tab) - 1)]


def _case(seed, *, q_lens, past, Hq, Hkv, D, Dp=None, page_size=32, rope=None, neox=True, src=BF16, kv=None, pad_rows=0, pad_tokens=0,
          table_rows=None, extra_heads=0, positions=None):
    rng = np.random.default_rng(seed)
    kv, rope, Dp = src if kv is None else kv, D if rope is None else rope, D if Dp is None else Dp
    ctx, bt, qsl, ns, T, P = batch(rng, q_lens, past, page_size, pad_rows, pad_tokens)
    c = dict(ctx=ctx, bt=bt, qsl=qsl, ns=ns, T=T, P=P, Hq=Hq, Hkv=Hkv, D=D, Dp=Dp, pg=page_size, rope=rope, neox=neox, src=src, kv=kv)
    c["tab"] = table(table_rows or int(max(ctx.max(), 1)), rope)
    c["q"], c["k"], c["v"] = (_inputs(rng, T, h, D, src) for h in (Hq, Hkv, Hkv))
    c["pos"] = token_positions(ctx, qsl, int(ns[0]), T)
    c["positions"] = None if positions is None else rng.integers(0, positions, T).astype(np.int32)
    c["C"] = 2 * Hkv + extra_heads
    c["live"] = c["pos"] > -10 ** 8
    turn = _rows(c["tab"], c["pos"], c["positions"])
    c["q32"], c["k32"] = (rotate(c[n][1], turn, rope, neox) for n in ("q", "k"))
    c["turn"] = turn
    return c


def _args(c, gpu):
    up = lambda n: tl.to_torch(c[n][0], c["src"], gpu)  # noqa: E731
    meta = [dev(c[n], gpu) for n in ("tab", "ctx", "bt", "qsl", "ns")]
    return up("q"), up("k"), up("v"), meta


def _want_queries(c):
    want = encode(c["q32"], c["src"])
    want[~c["live"]] = 0
    return want


def _check_queries(c, got, live_only=False):
    want = _want_queries(c)
    raw = raw_of(got, c["src"])
    if live_only:
        raw, want = raw[c["live"]], want[c["live"]]
    assert np.array_equal(raw, want)


def _stale(c, shape):
    return np.full(shape, STALE[c["kv"]])


def _want_pages(c, pool):
    k, v = (encode(x, c["kv"]) for x in (c["k32"], c["v"][1]))
    if c["kv"] == c["src"]:
        v = c["v"][0]
    out = pool.copy()
    wide = lambda x: np.concatenate([x, np.zeros((*x.shape[:2], c["Dp"] - c["D"]), x.dtype)], -1)  # noqa: E731
    return orc.page_scatter_ragged_ref(wide(k), wide(v), out, c["ctx"], c["bt"], c["qsl"], c["ns"])


SHAPES = [
    dict(q_lens=[1], past=[0], Hq=4, Hkv=2, D=128),                                                    # the first token of all
    dict(q_lens=[1, 1, 1], past=[31, 32, 700], Hq=32, Hkv=8, D=128, page_size=64),                     # decode rows at page borders
    dict(q_lens=[40, 1, 0, 33, 65], past=[5, 99, 12, 0, 63], Hq=8, Hkv=8, D=64, pad_rows=3, pad_tokens=4),  # an empty row, padding
    dict(q_lens=[7, 130], past=[3, 1], Hq=5, Hkv=1, D=80, Dp=128, rope=40, neox=False, page_size=16),  # stored padded, half turns
    dict(q_lens=[9, 2], past=[0, 15], Hq=6, Hkv=2, D=96, Dp=128, rope=24, page_size=16, extra_heads=2),  # heads nobody writes
    dict(q_lens=[3, 5], past=[2, 8], Hq=3, Hkv=3, D=20, rope=6, page_size=5),                          # groups of one element
    dict(q_lens=[11], past=[250], Hq=2, Hkv=1, D=256, rope=256, neox=False, page_size=128, pad_tokens=1),
    dict(q_lens=[6, 4], past=[-3, 10], Hq=4, Hkv=2, D=64),                                             # tokens ahead of position 0
    dict(q_lens=[30, 1], past=[0, 40], Hq=4, Hkv=2, D=128, table_rows=20),                             # rows clamped into the table
    dict(q_lens=[30, 1], past=[9, 40], Hq=4, Hkv=2, D=128, positions=4000, table_rows=3000),           # explicit rows
]


@pytest.mark.parametrize("src,kv", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, FP8), (F32, BF16), (BF16, F32), (F16, FP8)])
@pytest.mark.parametrize("n", range(len(SHAPES)))
def test_interleaved_pages_bit_for_bit(gpu, n, src, kv):
    c = _case(n, src=src, kv=kv, **SHAPES[n])
    q, k, v, meta = _args(c, gpu)
    pool = _stale(c, (c["P"], c["pg"], c["C"], c["Dp"]))
    pages = tl.to_torch(pool, kv, gpu)
    pos = None if c["positions"] is None else dev(c["positions"], gpu)
    got, same = kernels.rope_page_scatter_ragged(q, k, v, pages, *meta, is_neox_style=c["neox"], positions=pos)
    torch.cuda.synchronize()
    assert same is pages
    _check_queries(c, got)
    assert np.array_equal(raw_of(pages, kv), _want_pages(c, pool))


@pytest.mark.parametrize("src,kv", [(BF16, BF16), (F16, F16), (F32, F32), (F32, FP8)])
@pytest.mark.parametrize("with_count", [True, False])
@pytest.mark.parametrize("n", [2, 5, 6])
def test_separate_pools_bit_for_bit(gpu, n, with_count, src, kv):
    shape = {k: v for k, v in SHAPES[n].items() if k not in ("Dp", "extra_heads")}
    c = _case(50 + n, src=src, kv=kv, **shape)
    q, k, v, (tab, ctx, bt, qsl, ns) = _args(c, gpu)
    pool = _stale(c, (c["P"], c["pg"], c["Hkv"], c["D"]))
    kc, vc = tl.to_torch(pool, kv, gpu), tl.to_torch(pool, kv, gpu)
    got, _, _ = kernels.rope_unified_page_scatter(q, k, v, kc, vc, tab, ctx, bt, qsl, ns if with_count else None, is_neox_style=c["neox"])
    torch.cuda.synchronize()
    _check_queries(c, got)
    want = _want_pages(c, _stale(c, (c["P"], c["pg"], 2 * c["Hkv"], c["D"])))
    assert np.array_equal(raw_of(kc, kv), want[:, :, 0::2]) and np.array_equal(raw_of(vc, kv), want[:, :, 1::2])


@pytest.mark.parametrize("kv", [FP8, INT8])
@pytest.mark.parametrize("src", [BF16, F32, F16])
@pytest.mark.parametrize("D,Dp,rope,neox,pg,Hkv", [(128, 128, 128, True, 64, 4), (64, 64, 32, False, 16, 2), (80, 128, 80, True, 32, 3), (20, 20, 12, True, 5, 1)])
def test_scaled_pages_bit_for_bit_over_serving_steps(gpu, kv, src, D, Dp, rope, neox, pg, Hkv):
    # prompts, chunks and decode steps on the same pages: fresh pages ignore their stale scales, scales grow, old codes change
    rng = np.random.default_rng(7 * D + kv)
    S, M, P, Hq = 5, 6, 40, 2 * Hkv
    bt = rng.permutation(np.arange(1, P)).astype(np.int32)[:S * M].reshape(S, M)
    codes = rng.integers(0, 120, size=(P, pg, 2 * Hkv, Dp), dtype=np.uint8)
    codes[..., D:] = 0
    scales = rng.uniform(0.5, 4.0, size=(P, 2 * Hkv)).astype(np.float32)
    tab = table(M * pg, rope)
    ctx = np.zeros(S, np.int32)
    for step, q_lens in enumerate([[pg + 5, 3, 1, 2 * pg, 0], [1, pg - 3, 1, 7, 9], [1, 1, 1, 1, 1], [1, 1, 0, 1, 1], [3, 1, 1, 1, pg]]):
        q_lens = np.array(q_lens, np.int32)
        ctx = (ctx + q_lens).astype(np.int32)
        qsl = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        T, live = int(qsl[-1]) + 2, np.where(q_lens > 0, ctx, 0).astype(np.int32)
        gain = 1.0 + 0.6 * step
        (q_raw, q32), (k_raw, k32), (v_raw, v32) = ((encode((x * gain).astype(np.float32), src), None) for x in
                                                    (rng.standard_normal((T, h, D)) for h in (Hq, Hkv, Hkv)))
        q32, k32, v32 = (decode(r, src) for r in (q_raw, k_raw, v_raw))
        turn = _rows(tab, token_positions(live, qsl, S, T))
        k_turned = rotate(k32, turn, rope, neox)
        want_codes, want_scales = append_scaled(k_turned, v32, codes[..., :D], scales, live, bt, qsl, S, kv)
        pages = dev(codes, gpu).view(torch.float8_e4m3fn if kv == FP8 else torch.int8)
        sc = dev(scales, gpu)
        got, _, _ = kernels.rope_page_scatter_ragged(*(tl.to_torch(r, src, gpu) for r in (q_raw, k_raw, v_raw)), pages, dev(tab, gpu), dev(live, gpu),
                                                     dev(bt, gpu), dev(qsl, gpu), dev(np.array([S], np.int32), gpu), kv_scales=sc, is_neox_style=neox)
        torch.cuda.synchronize()
        codes, scales = pages.view(torch.uint8).cpu().numpy(), sc.cpu().numpy()
        assert np.array_equal(scales, want_scales), step
        assert np.array_equal(codes[..., :D], want_codes), step
        assert not codes[..., D:].any()
        want_q = encode(rotate(q32, turn, rope, neox), src)
        want_q[qsl[-1]:] = 0
        assert np.array_equal(raw_of(got, src), want_q), step


LATENT = [dict(q_lens=[1], past=[0], Hq=2, lkv=64, rope=64), dict(q_lens=[1, 1, 40, 0], past=[63, 64, 20, 5], Hq=16, lkv=512, rope=64, neox=False, pad_tokens=3),
          dict(q_lens=[5, 17], past=[2, 30], Hq=7, lkv=72, rope=24, pad_rows=2), dict(q_lens=[9], past=[-4], Hq=128, lkv=512, rope=128, neox=False),
          dict(q_lens=[3], past=[1], Hq=1, lkv=8, rope=8)]


@pytest.mark.parametrize("src,kv", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, FP8), (F32, BF16)])
@pytest.mark.parametrize("n", range(len(LATENT)))
def test_latent_pages_bit_for_bit(gpu, n, src, kv):
    sh = dict(LATENT[n])
    lkv, rope, Hq, neox = sh.pop("lkv"), sh.pop("rope"), sh.pop("Hq"), sh.pop("neox", True)
    rng = np.random.default_rng(300 + n)
    pg = 64
    ctx, bt, qsl, ns, T, P = batch(rng, sh.pop("q_lens"), sh.pop("past"), pg, **sh)
    tab = table(int(max(ctx.max(), 1)), rope)
    (q_raw, q32), (k_raw, k32) = _inputs(rng, T, Hq, rope, src), _inputs(rng, T, 1, rope, src)
    kv_raw, _ = _inputs(rng, T, 1, lkv, kv)
    row = -(-lkv // 128) * 128 + -(-rope // 128) * 128
    pool = np.full((P, pg, row), STALE[kv])
    pages = tl.to_torch(pool, kv, gpu)
    pos = token_positions(ctx, qsl, int(ns[0]), T)
    turn = _rows(tab, pos)
    got, _ = kernels.rope_mla_page_scatter(tl.to_torch(q_raw, src, gpu), tl.to_torch(kv_raw[:, 0], kv, gpu), tl.to_torch(k_raw[:, 0], src, gpu), pages,
                                           dev(tab, gpu), dev(ctx, gpu), dev(bt, gpu), dev(qsl, gpu), dev(ns, gpu), is_neox_style=neox)
    torch.cuda.synchronize()
    want_q = encode(rotate(q32, turn, rope, neox), src)
    want_q[pos < -10 ** 8] = 0
    assert np.array_equal(raw_of(got, src), want_q)
    pe = encode(rotate(k32, turn, rope, neox), kv)[:, 0]
    assert np.array_equal(raw_of(pages, kv), orc.mla_page_scatter_ref(kv_raw[:, 0], pe, pool, ctx, bt, qsl, ns))


@pytest.mark.parametrize("src,unit", [(BF16, 2.0 ** -8), (F16, 2.0 ** -11), (F32, 0.0)])
@pytest.mark.parametrize("neox", [True, False])
def test_rotation_against_64_bits(gpu, src, unit, neox):
    """Each of the two products and the sum is off by at most half a float32 step (2^-24 of itself), the result by half a
    step of its type: |error| <= unit |y| + (1 + unit) 2 * 2^-24 (|a c| + |b s|), |a c| + |b s| <= |a| + |b| =: m, and half of the
    smallest subnormal of half precision."""
    c = _case(77, q_lens=[50, 1], past=[30, 5000], Hq=4, Hkv=2, D=128, rope=96, neox=neox, src=src)
    q, k, v, meta = _args(c, gpu)
    pages = torch.zeros((c["P"], c["pg"], c["C"], c["Dp"]), dtype=q.dtype, device=gpu)
    got, _ = kernels.rope_page_scatter_ragged(q, k, v, pages, *meta, is_neox_style=neox)
    torch.cuda.synchronize()
    y = rotate(c["q"][1], c["turn"], 96, neox, np.float64)
    m = np.abs(c["q"][1].astype(np.float64))
    both = m[..., :96].reshape(*m.shape[:2], 2, 48).sum(2) if neox else m[..., :96].reshape(*m.shape[:2], 48, 2).sum(3)
    m[..., :96] = np.concatenate([both, both], -1) if neox else np.repeat(both, 2, -1)
    err = np.abs(tl.from_torch(got, src) - y)
    assert (err <= unit * np.abs(y) + 1.01 * 2 * 2.0 ** -24 * m + (2.0 ** -25 if src == F16 else 0.0)).all()


def test_views_of_one_projection(gpu):
    c = _case(5, q_lens=[20, 1], past=[3, 40], Hq=4, Hkv=2, D=64)
    q, k, v, meta = _args(c, gpu)
    T = c["T"]
    pool = _stale(c, (c["P"], c["pg"], c["C"], c["Dp"]))
    want = _want_pages(c, pool)
    for lead in (0, 8, 1):  # the second projection's rows are aligned to 16 bytes, the third's to nothing but their elements
        qkv = torch.cat([torch.full((T, lead), 3.0, dtype=q.dtype, device=gpu), q.flatten(1), k.flatten(1), v.flatten(1)], dim=1)
        views = [x.unflatten(1, (-1, 64)) for x in qkv[:, lead:].split((256, 128, 128), dim=1)]
        pages = tl.to_torch(pool, BF16, gpu)
        got, _ = kernels.rope_page_scatter_ragged(*views, pages, *meta)
        torch.cuda.synchronize()
        _check_queries(c, got)
        assert np.array_equal(raw_of(pages, BF16), want)


def test_in_place_leaves_padded_rows(gpu):
    c = _case(6, q_lens=[20, 1], past=[3, 40], Hq=4, Hkv=2, D=64, pad_tokens=3)
    q, k, v, meta = _args(c, gpu)
    before = q.clone()
    pages = tl.to_torch(_stale(c, (c["P"], c["pg"], c["C"], c["Dp"])), BF16, gpu)
    got, _ = kernels.rope_page_scatter_ragged(q, k, v, pages, *meta, query_out=q)
    torch.cuda.synchronize()
    assert got is q
    _check_queries(c, got, live_only=True)
    assert torch.equal(q[c["T"] - 3:], before[c["T"] - 3:])


def test_bare_fp8_cast_at_its_borders(gpu):
    """448 is kept, 464 is the tie that goes to 448, beyond it NaN; zeros keep their sign; subnormals round to even."""
    v = np.array([448, 463.9, 464, 464.1, 480, 1e9, np.inf, -448, -464, -465, -np.inf, np.nan, 0.0, -0.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 2.5 * 2.0 ** -9,
                  2.0 ** -10 * 1.01, 17.0, 18.0, 19.0, 1.0625, 1.1875], np.float32)
    D = 24
    k = torch.zeros((1, 1, D), device=gpu)
    pages = torch.zeros((1, 1, 2, D), dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)
    one = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    kernels.rope_page_scatter_ragged(k, k.clone(), torch.from_numpy(v).to(gpu).reshape(1, 1, D), pages, torch.ones((1, 2), device=gpu), one(1), one(0), one(0, 1), one(1))
    torch.cuda.synchronize()
    got, want = pages.view(torch.uint8)[0, 0, 1].cpu(), torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(got, want)


def test_bad_pages_and_foreign_rows_are_left_alone(gpu):
    """Page ids outside the pool and positions behind the block table are dropped; so are rows of the pool nobody owns."""
    c = _case(8, q_lens=[40, 3], past=[10, 5], Hq=4, Hkv=2, D=64, page_size=16)
    q, k, v, (tab, ctx, bt, qsl, ns) = _args(c, gpu)
    pool = _stale(c, (c["P"], 16, 4, 64))
    want = _want_pages(c, pool)
    lost = c["bt"][0, 1:3].copy()
    bt_bad = c["bt"].copy()
    bt_bad[0, 1], bt_bad[0, 2] = -1, c["P"]
    want[lost] = pool[lost]
    pages = tl.to_torch(pool, BF16, gpu)
    got, _ = kernels.rope_page_scatter_ragged(q, k, v, pages, tab, ctx, dev(bt_bad, gpu), qsl, ns)
    torch.cuda.synchronize()
    assert np.array_equal(raw_of(pages, BF16), want)
    _check_queries(c, got)
    codes = torch.zeros((c["P"], 16, 4, 64), dtype=torch.int8, device=gpu)
    scales = torch.full((c["P"], 4), 2.0, device=gpu)
    kernels.rope_page_scatter_ragged(q, k, v, codes, tab, ctx, dev(bt_bad, gpu), qsl, ns, kv_scales=scales)
    torch.cuda.synchronize()
    untouched = np.setdiff1d(np.arange(c["P"]), [p for i, n in enumerate(c["ctx"]) for p in bt_bad[i, (int(n) - [40, 3][i]) // 16:-(-int(n) // 16)]])
    assert not codes[untouched].any() and (scales[untouched] == 2.0).all()
    short = dev(c["bt"][:, :2], gpu)  # the first sequence's last two pages have no column
    pages = tl.to_torch(pool, BF16, gpu)
    got, _ = kernels.rope_page_scatter_ragged(q, k, v, pages, tab, ctx, short, qsl, ns)
    torch.cuda.synchronize()
    want = _want_pages(c, pool)
    want[c["bt"][0, 2:4]] = pool[c["bt"][0, 2:4]]
    assert np.array_equal(raw_of(pages, BF16), want)


def test_replayed_from_a_graph_and_on_another_stream(gpu):
    c = _case(9, q_lens=[20, 1], past=[3, 40], Hq=4, Hkv=2, D=128)
    q, k, v, meta = _args(c, gpu)
    pool = tl.to_torch(_stale(c, (c["P"], c["pg"], c["C"], c["Dp"])), BF16, gpu)
    pages, out = pool.clone(), torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.rope_page_scatter_ragged(q, k, v, pages, *meta, query_out=out)
    torch.cuda.current_stream().wait_stream(side)
    want = pages.clone()
    _check_queries(c, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.rope_page_scatter_ragged(q, k, v, pages, *meta, query_out=out)
    for _ in range(3):
        pages.copy_(pool)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pages, want)
        _check_queries(c, out)


def test_a_long_pool_past_32_bit_offsets(gpu):
    """Rows beyond 2^32 bytes of the pool (40 000 pages of 256 KiB)."""
    c = _case(11, q_lens=[20, 1], past=[3, 40], Hq=4, Hkv=8, D=128, page_size=64)
    q, k, v, (tab, ctx, bt, qsl, ns) = _args(c, gpu)
    far = c["bt"].copy()
    far[far >= 0] += 39_000
    pages = torch.zeros((40_000, 64, 16, 128), dtype=torch.bfloat16, device=gpu)
    kernels.rope_page_scatter_ragged(q, k, v, pages, tab, ctx, dev(far, gpu), qsl, ns)
    torch.cuda.synchronize()
    want = _want_pages(c, np.zeros((c["P"], 64, 16, 128), np.uint16))
    assert np.array_equal(raw_of(pages[39_000:39_000 + c["P"]], BF16), want)
    assert not pages[:39_000].any()
