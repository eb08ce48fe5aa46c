"""GPU tests of linear attention with a decay per head, against the recurrence in 64 bits.

Tolerance: with A_t = l A_{t-1} + |k_t| |v_t|^T (what the state could be at most) every float32 sum of n terms is off by at most
about n 2^-24 of the sum of its terms' sizes, and the decay powers by 2^-24 each, so a state is off by less than
(2 n + 2 Dk + 64) 2^-24 A and an output by that times |q|, plus half a step of its type.  Inputs of 16 bits also allow the two
operands that meet the matrix instructions as rounded 16-bit values, the scores inside a chunk and the state it starts from:
half a bfloat16 step (2^-8) of each term.  Sums of the sizes themselves are taken in 64 bits."""

import numpy as np
import pytest
import torch

from easydel_amd import kernels
from rope_testlib import BF16, F16, F32, decode, dev, encode, tl

pytestmark = pytest.mark.gpu

UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TORCH = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}


class Case:
    pass


def make(seed, q_lens, *, Hq=4, Hkv=4, Dk=64, Dv=64, tag=BF16, past=None, pad_rows=0, pad_tokens=0, decays=None, slots=None, spare=2, gain=1.0):
    rng = np.random.default_rng(seed)
    c = Case()
    c.Hq, c.Hkv, c.Dk, c.Dv, c.tag, c.n = Hq, Hkv, Dk, Dv, tag, len(q_lens)
    c.q_lens = np.asarray(q_lens, np.int32)
    c.S = c.n + pad_rows
    c.qsl = np.zeros(c.S + 1, np.int32)
    c.qsl[1:c.n + 1] = np.cumsum(c.q_lens)
    c.qsl[c.n + 1:] = c.qsl[c.n]
    c.T = int(c.qsl[c.n]) + pad_tokens
    c.past = np.asarray([10] * c.n if past is None else past, np.int32)
    c.ctx = np.zeros(c.S, np.int32)
    c.ctx[:c.n] = c.q_lens + c.past
    enc = lambda *shape: encode((rng.standard_normal(shape) * gain).astype(np.float32), tag)  # noqa: E731
    c.q, c.k, c.v = enc(c.T, Hq, Dk), enc(c.T, Hkv, Dk), enc(c.T, Hkv, Dv)
    c.log_decay = (-np.exp(rng.uniform(np.log(1e-3), 0.0, Hkv)) if decays is None else np.resize(decays, Hkv)).astype(np.float32)
    c.N = slots or 2 * c.S + spare
    c.state = rng.standard_normal((c.N, Hkv, Dk, Dv)).astype(np.float32)
    perm = rng.permutation(c.N)[:2 * c.S].astype(np.int32) if 2 * c.S <= c.N else np.zeros(2 * c.S, np.int32)
    c.slot_in, c.slot_out = perm[:c.S].copy(), perm[c.S:].copy()
    return c


def oracle(c, in_place=False):
    """(out, its size bound, state, its size bound): 64 bits, token by token; rows of padded tokens are zeros."""
    q, k, v = (decode(x, c.tag).astype(np.float64) for x in (c.q, c.k, c.v))
    lam = np.exp(c.log_decay.astype(np.float64))[:, None, None]
    G = c.Hq // c.Hkv
    out, size = np.zeros((c.T, c.Hq, c.Dv)), np.zeros((c.T, c.Hq, c.Dv))
    state = c.state.astype(np.float64)
    bound = np.zeros_like(state)
    scale = c.Dk ** -0.5
    for i in range(c.n):
        if c.q_lens[i] == 0:
            continue
        a = int(c.slot_in[i])
        S = c.state[a].astype(np.float64) if c.past[i] > 0 and 0 <= a < c.N else np.zeros((c.Hkv, c.Dk, c.Dv))
        A = np.abs(S)
        for t in range(c.qsl[i], c.qsl[i + 1]):
            S = lam * S + k[t][:, :, None] * v[t][:, None, :]
            A = lam * A + np.abs(k[t][:, :, None] * v[t][:, None, :])
            out[t] = scale * np.matmul(q[t].reshape(c.Hkv, G, c.Dk), S).reshape(c.Hq, c.Dv)
            size[t] = scale * np.matmul(np.abs(q[t]).reshape(c.Hkv, G, c.Dk), A).reshape(c.Hq, c.Dv)
        b = int(c.slot_in[i] if in_place else c.slot_out[i])
        if 0 <= b < c.N:
            state[b], bound[b] = S, A
    return out, size, state, bound


def upload(c, gpu):
    up = lambda x: tl.to_torch(x, c.tag, gpu)  # noqa: E731
    return dict(q=up(c.q), k=up(c.k), v=up(c.v), g=dev(c.log_decay, gpu), state=dev(c.state, gpu), slot_in=dev(c.slot_in, gpu),
                slot_out=dev(c.slot_out, gpu), ctx=dev(c.ctx, gpu), qsl=dev(c.qsl, gpu), ns=dev(np.array([c.n], np.int32), gpu))


def call(d, in_place=False, **kw):
    return kernels.decay_linear_attention(d["q"], d["k"], d["v"], d["g"], d["state"], d["slot_in"], d["qsl"], d["ns"], context_lens=d["ctx"],
                                          state_out_indices=None if in_place else d["slot_out"], **kw)


def check(c, out, state, in_place=False):
    want, size, want_state, bound = oracle(c, in_place)
    n = max(int(c.q_lens.max()), 1)
    steps = (2 * n + 2 * c.Dk + 64) * 2.0 ** -24
    got, got_state = tl.from_torch(out, c.tag), state.cpu().numpy().astype(np.float64)
    unit = UNIT[c.tag]
    halves = 0.0 if c.tag == F32 else 2.0 ** -8
    tiny = 2.0 ** -25 if c.tag == F16 else 0.0
    err = np.abs(got - want)
    assert (err <= unit * np.abs(want) + (1 + unit) * (steps + halves) * size + tiny).all(), (err - unit * np.abs(want)).max()
    assert (np.abs(got_state - want_state) <= steps * bound).all()  # slots nobody writes: bound 0, equal bit for bit
    # as a whole the errors are roundings, not faults: with every term off by half a step of its own the 2-norm stays near one step
    if want.any():
        assert np.linalg.norm(got - want) <= max(1.5 * unit, 4e-6) * np.linalg.norm(want)


SHAPES = [
    dict(q_lens=[1]),
    dict(q_lens=[1] * 9, Hq=8, Hkv=2, Dk=128, Dv=128, past=[0, 1, 5, 0, 7, 9, 1, 0, 3], pad_rows=2, pad_tokens=3),
    dict(q_lens=[2, 0, 17, 1, 64, 65], Hq=4, Hkv=4, Dk=128, Dv=128, past=[0, 4, 4, 4, 0, 9], pad_rows=1, pad_tokens=5),
    dict(q_lens=[63, 128, 129, 5], Hq=6, Hkv=2, Dk=64, Dv=96),
    dict(q_lens=[700, 3], Hq=2, Hkv=1, Dk=256, Dv=200, past=[0, 2]),
    dict(q_lens=[1500, 40], Hq=2, Hkv=2, Dk=128, Dv=64),
    dict(q_lens=[33, 90], Hq=3, Hkv=3, Dk=20, Dv=12, pad_tokens=1),
    dict(q_lens=[300, 16, 15, 17], Hq=2, Hkv=2, Dk=128, Dv=256, past=[1, 0, 1, 1]),
    dict(q_lens=[130, 70], Hq=2, Hkv=2, Dk=4, Dv=4),
    dict(q_lens=[200, 1], Hq=2, Hkv=2, Dk=72, Dv=136),
]


@pytest.mark.parametrize("tag", [BF16, F32, F16])
@pytest.mark.parametrize("n", range(len(SHAPES)))
def test_against_the_recurrence_in_64_bits(gpu, n, tag):
    c = make(n, tag=tag, **SHAPES[n])
    d = upload(c, gpu)
    out, state = call(d)
    torch.cuda.synchronize()
    assert state is d["state"] and out.dtype == TORCH[tag]
    check(c, out, state)
    if c.T > c.qsl[c.n]:
        assert not out[int(c.qsl[c.n]):].any()


@pytest.mark.parametrize("tag", [BF16, F32])
@pytest.mark.parametrize("decays", [[0.0], [-np.inf], [-1e-6, -100.0], [-30.0, -0.5], [-3e38]])
def test_decays_at_their_ends(gpu, tag, decays):
    c = make(40, [150, 1, 20], Hq=2, Hkv=2, Dk=128, Dv=64, tag=tag, decays=np.array(decays), past=[3, 3, 0])
    d = upload(c, gpu)
    out, state = call(d)
    torch.cuda.synchronize()
    check(c, out, state)


@pytest.mark.parametrize("tag", [BF16, F32])
def test_in_place_and_step_by_step(gpu, tag):
    """A prompt in one call, in two calls, and token by token through the same slots."""
    c = make(50, [90, 75], Hq=4, Hkv=2, Dk=128, Dv=128, tag=tag, past=[0, 6])
    d = upload(c, gpu)
    start = d["state"].clone()
    out, state = call(d, in_place=True)
    check(c, out, state, in_place=True)
    whole = state.clone()
    for cuts in ([0, 41], [0] + list(range(60, 75))):
        d["state"] = start.clone()
        parts = [[], []]
        for a, b in zip(cuts, cuts[1:] + [None]):
            ends = [n if b is None else b for n in c.q_lens]
            rows = [slice(int(c.qsl[i]) + a, int(c.qsl[i]) + e) for i, e in enumerate(ends)]
            lens = [e - a for e in ends]
            piece = dict(d, q=torch.cat([d["q"][r] for r in rows]), k=torch.cat([d["k"][r] for r in rows]), v=torch.cat([d["v"][r] for r in rows]),
                         qsl=dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), gpu), ctx=dev((c.past + ends).astype(np.int32), gpu))
            got, _ = call(piece, in_place=True)
            parts[0].append(got[:lens[0]])
            parts[1].append(got[lens[0]:])
        torch.cuda.synchronize()
        check(c, torch.cat(parts[0] + parts[1]), d["state"], in_place=True)
    assert torch.isfinite(whole).all()


@pytest.mark.parametrize("group", [2, 4, 7])
@pytest.mark.parametrize("tail", [1, 5, 16, 17, 31])
def test_last_chunks_of_shared_heads(gpu, group, tail):
    """Several query heads a KV head in a last chunk that is not full: each head's queries are waited for although the stores of the
    head before were fewer.  Many sequences, so that the loads are slow."""
    c = make(54 + tail, [32 + tail] * 64, Hq=2 * group, Hkv=2, Dk=128, Dv=128)
    d = upload(c, gpu)
    out, state = call(d)
    out, state = out.clone(), state.clone()
    check(c, out, state)
    for _ in range(5):
        again, _ = call(d)
        torch.cuda.synchronize()
        assert torch.equal(out, again) and torch.equal(state, d["state"])


@pytest.mark.parametrize("tag", [BF16, F32])
def test_cut_prompts_in_place(gpu, tag):
    """Sequences long enough to be cut into segments that run side by side: the slot they start from is the slot they end in."""
    c = make(51, [1700, 1, 300, 900], Hq=4, Hkv=2, Dk=128, Dv=64, tag=tag, past=[4, 4, 4, 0])
    d = upload(c, gpu)
    for _ in range(3):
        d["state"] = dev(c.state, gpu)
        out, state = call(d, in_place=True)
        torch.cuda.synchronize()
        check(c, out, state, in_place=True)


def test_workspace_of_cut_prompts(gpu):
    """A call that cuts its prompts refuses a workspace below the size it asks for, and needs none where nothing can be cut."""
    from easydel_amd import _lib

    lib = _lib.load()
    assert lib.rpa_decay_attention_workspace_bytes(16, 4, 8, 8, 128, 128, 1) == 0
    need = lib.rpa_decay_attention_workspace_bytes(1700, 1, 4, 2, 128, 64, 1)
    assert need > 0
    c = make(52, [1700], Hq=4, Hkv=2, Dk=128, Dv=64)
    d = upload(c, gpu)
    out = torch.full((c.T, 4, 64), 7.0, dtype=torch.bfloat16, device=gpu)
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    args = lambda w, n: (torch.cuda.current_stream().cuda_stream, d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(), d["g"].data_ptr(),  # noqa: E731
                         d["state"].data_ptr(), d["slot_in"].data_ptr(), d["slot_out"].data_ptr(), d["ctx"].data_ptr(), d["qsl"].data_ptr(),
                         d["ns"].data_ptr(), out.data_ptr(), w, n, c.T, c.S, c.N, 4, 2, 128, 64, 512, 256, 128, 1, 128 ** -0.5)
    assert lib.rpa_decay_linear_attention(*args(ws.data_ptr(), need - 1)) == _lib.RPA_ERR_WORKSPACE
    assert lib.rpa_decay_linear_attention(*args(None, need)) == _lib.RPA_ERR_WORKSPACE
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    assert lib.rpa_decay_linear_attention(*args(ws.data_ptr(), need)) == 0
    torch.cuda.synchronize()
    check(c, out, d["state"])


def test_slots(gpu):
    """Two sequences read one slot (a shared prefix); slots outside the pool read as zeros and are not written."""
    c = make(60, [5, 80, 1, 70], Hq=2, Hkv=2, Dk=64, Dv=64)
    c.slot_in[:4] = [3, 3, -1, c.N]
    c.slot_out[:4] = [0, 1, c.N + 5, -7]
    d = upload(c, gpu)
    out, state = call(d)
    torch.cuda.synchronize()
    check(c, out, state)


def test_without_context_lens_every_sequence_goes_on(gpu):
    c = make(61, [5, 80], past=[0, 0])
    d = upload(c, gpu)
    out, state = kernels.decay_linear_attention(d["q"], d["k"], d["v"], d["g"], d["state"], d["slot_in"], d["qsl"], d["ns"], state_out_indices=d["slot_out"])
    torch.cuda.synchronize()
    c.past[:] = 1
    check(c, out, state)


@pytest.mark.parametrize("tag", [BF16, F32, F16])
def test_garbage_stays_where_it_is(gpu, tag):
    """NaN in a fresh sequence's slot, in padded rows, and in one sequence's tokens: none of it reaches another sequence, nor a
    token ahead of it in its own."""
    c = make(62, [70, 1, 90, 3, 130], Hq=2, Hkv=2, Dk=128, Dv=64, tag=tag, past=[0, 5, 5, 0, 0], pad_tokens=4)
    d = upload(c, gpu)
    clean, clean_state = call(d)
    clean, clean_state = clean.clone(), clean_state.clone()
    d = upload(c, gpu)
    for i in (0, 3, 4):
        d["state"][int(c.slot_in[i])] = float("nan")
    bad = int(c.qsl[2]) + 37  # inside the third sequence
    for x in ("q", "k", "v"):
        d[x][c.T - 4:] = float("nan")
    d["k"][bad, 0, 5] = float("inf")
    d["v"][bad, 0, 7] = float("nan")
    d["v"][bad, 1, 3] = float("inf")
    out, state = call(d)
    torch.cuda.synchronize()
    hurt = torch.zeros(c.T, dtype=torch.bool, device=gpu)
    hurt[bad:int(c.qsl[3])] = True
    assert torch.equal(out[~hurt], clean[~hurt])
    assert not torch.isfinite(out[bad:int(c.qsl[3]), 0, 7]).any()
    third = int(c.slot_out[2])
    keep = [i for i in range(c.N) if i != third and i not in [int(c.slot_in[j]) for j in (0, 3, 4)]]
    assert torch.equal(state[keep], clean_state[keep])


def test_views_of_one_projection(gpu):
    for lead, tag in ((0, BF16), (1, BF16), (4, F32), (2, F32)):
        c = make(63, [100, 1, 30], Hq=4, Hkv=2, Dk=64, Dv=96, tag=tag)
        d = upload(c, gpu)
        qkv = torch.cat([torch.full((c.T, lead), 3.0, dtype=d["q"].dtype, device=gpu), d["q"].flatten(1), d["k"].flatten(1), d["v"].flatten(1)], dim=1)
        q, k, v = qkv[:, lead:].split((256, 128, 192), dim=1)
        d.update(q=q.unflatten(1, (4, 64)), k=k.unflatten(1, (2, 64)), v=v.unflatten(1, (2, 96)))
        out, state = call(d)
        torch.cuda.synchronize()
        check(c, out, state)


def test_replayed_from_a_graph_with_eager_calls_between(gpu):
    c = make(64, [600, 1, 40], Hq=4, Hkv=4, Dk=128, Dv=128)
    d = upload(c, gpu)
    out = torch.empty((c.T, 4, 128), dtype=torch.bfloat16, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(d, out=out)
    torch.cuda.current_stream().wait_stream(side)
    want, want_state = out.clone(), d["state"].clone()
    check(c, out, d["state"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(d, out=out)
    other = make(65, [2000, 3, 500], Hq=4, Hkv=4, Dk=128, Dv=128)
    e = upload(other, gpu)
    for _ in range(3):
        out.fill_(3.0)
        d["state"].copy_(dev(c.state, gpu))
        graph.replay()
        call(e)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(d["state"], want_state)


def test_the_same_call_twice_gives_the_same_bits(gpu):
    c = make(66, [900, 1, 333, 64], Hq=8, Hkv=4, Dk=128, Dv=128)
    d = upload(c, gpu)
    a, s = call(d)
    a, s = a.clone(), s.clone()
    for _ in range(3):
        b, _ = call(d)
        torch.cuda.synchronize()
        assert torch.equal(a, b) and torch.equal(s, d["state"])


def test_a_pool_past_32_bit_offsets(gpu):
    """Slots beyond 2^32 bytes (70 000 states of 64 KiB)."""
    c = make(67, [70, 1], Hq=1, Hkv=1, Dk=128, Dv=128)
    d = upload(c, gpu)
    small = d["state"]
    d["state"] = torch.zeros((70_000, 1, 128, 128), device=gpu)
    at = 70_000 - c.N
    d["state"][at:] = small
    d["slot_in"] += at
    d["slot_out"] += at
    out, state = call(d)
    torch.cuda.synchronize()
    check(c, out, state[at:])
    assert not state[:at].any()


def test_random_batches(gpu):
    for seed in range(24):
        rng = np.random.default_rng(900 + seed)
        Hkv = int(rng.choice([1, 2, 3]))
        lens = [int(x) for x in rng.choice([0, 1, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 200, 257], size=rng.integers(1, 7))]
        tag = [BF16, F32, F16][seed % 3]
        c = make(seed, lens, Hq=Hkv * int(rng.choice([1, 1, 2, 4])), Hkv=Hkv, Dk=int(rng.choice([16, 32, 64, 100, 128, 256])),
                 Dv=int(rng.choice([16, 32, 64, 72, 128, 160, 256])), tag=tag, past=rng.choice([0, 3], size=len(lens)), pad_rows=int(rng.integers(0, 3)),
                 pad_tokens=int(rng.integers(0, 3)) + (sum(lens) == 0))
        d = upload(c, gpu)
        out, state = call(d)
        torch.cuda.synchronize()
        check(c, out, state)


@pytest.mark.parametrize("tag", [BF16, F32])
def test_many_padded_rows(gpu, tag):
    """More metadata rows than the tokens could fill: segments are numbered by token instead of by row."""
    for lens, pad in (([17, 1, 0, 40, 18], 300), ([90], 200), ([700, 2, 33], 4000), ([1, 2], 64)):
        c = make(70, lens, Hq=4, Hkv=2, Dk=64, Dv=64, tag=tag, pad_rows=pad, pad_tokens=3, slots=2 * len(lens) + 2, past=[2] * len(lens))
        c.slot_in[:len(lens)] = np.arange(len(lens))
        c.slot_out[:len(lens)] = len(lens) + np.arange(len(lens))
        d = upload(c, gpu)
        out, state = call(d)
        torch.cuda.synchronize()
        check(c, out, state)
        assert not out[int(c.qsl[c.n]):].any()


def test_one_graph_serves_other_batches_of_its_bounds(gpu):
    """Lengths, slots and live rows are read by the kernels: a graph captured over one batch is replayed over others."""
    first = make(71, [600, 1, 40, 30], Hq=4, Hkv=2, Dk=128, Dv=128)
    d = upload(first, gpu)
    out = torch.empty((first.T, 4, 128), dtype=torch.bfloat16, device=gpu)
    call(d, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(d, out=out)
    for seed, lens, pad_rows in ((72, [1, 1, 1, 1], 0), (73, [671], 3), (74, [16, 17, 300, 0], 0), (75, [5, 650], 2), (71, [600, 1, 40, 30], 0)):
        c = make(seed, lens, Hq=4, Hkv=2, Dk=128, Dv=128, pad_rows=pad_rows, pad_tokens=first.T - sum(lens))
        for key, new in upload(c, gpu).items():
            d[key].copy_(new)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        check(c, out, d["state"])
        assert not out[int(c.qsl[c.n]):].any()


def test_two_streams_at_once(gpu):
    """Calls on two streams have scratch of their own."""
    cases = [make(76 + i, [1500, 3, 200], Hq=4, Hkv=2, Dk=128, Dv=128) for i in range(2)]
    data = [upload(c, gpu) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for c, d in zip(cases, data):
            d["state"].copy_(dev(c.state, gpu))
        torch.cuda.synchronize()
        outs = []
        for d, s in zip(data, streams):
            with torch.cuda.stream(s):
                outs.append(call(d)[0])
        torch.cuda.synchronize()
        for c, d, out in zip(cases, data, outs):
            check(c, out, d["state"])


def test_rows_far_apart(gpu):
    """Token rows 2^23 elements apart: offsets inside a chunk pass 31 bits."""
    c = make(79, [40, 3], Hq=1, Hkv=1, Dk=16, Dv=16)
    d = upload(c, gpu)
    wide = torch.zeros((c.T, 1 << 23), dtype=torch.bfloat16, device=gpu)
    for name, at in (("q", 0), ("k", 16), ("v", 32)):
        wide[:, at:at + 16] = d[name].flatten(1)
        d[name] = wide[:, at:at + 16].unflatten(1, (1, 16))
    out, state = call(d)
    torch.cuda.synchronize()
    check(c, out, state)


def test_no_tokens(gpu):
    c = make(80, [4], Hq=2, Hkv=2)
    d = upload(c, gpu)
    want = d["state"].clone()
    empty = dict(d, q=d["q"][:0], k=d["k"][:0], v=d["v"][:0])
    out, state = call(empty)
    assert tuple(out.shape) == (0, 2, 64) and torch.equal(state, want)
    d["ns"].zero_()
    out, state = call(d)  # no live row: outputs are zeros, states as they were
    torch.cuda.synchronize()
    assert not out.any() and torch.equal(state, want)


def test_scratch_starts_where_the_wrapper_asks_for_it(gpu):
    """The library cuts nothing in calls of up to as many tokens as the wrapper does not ask for; calls around that border run."""
    from easydel_amd import _lib

    lib, whole = _lib.load(), kernels._DECAY_WHOLE
    sizes = [(S, Hkv, dk, dv) for S in (1, 7, 4000) for Hkv in (1, 2, 64) for dk, dv in ((4, 4), (128, 128), (256, 256))]
    need = lambda T: [lib.rpa_decay_attention_workspace_bytes(T, S, Hkv, Hkv, dk, dv, 1) for S, Hkv, dk, dv in sizes]  # noqa: E731
    for T in (1, 16, 17, 100, whole - 1, whole):
        assert not any(need(T))
    assert any(need(whole + 1))
    for T in (whole - 1, whole, whole + 1, whole + 2):
        c = make(90, [T], Hq=1, Hkv=1, Dk=64, Dv=64)
        d = upload(c, gpu)
        out, state = call(d)
        torch.cuda.synchronize()
        check(c, out, state)
