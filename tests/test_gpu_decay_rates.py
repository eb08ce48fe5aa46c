"""GPU tests of linear attention with a decay per head over the whole range of decays, against the recurrence in 64 bits.

Every KV head has a decay of its own, from none at all to one that keeps nothing, with the band between log decays of -2.73 and
-3.25 whose power over a chunk of 32 tokens is a float32 subnormal.

Tolerance: that of the decayed attention's other tests, but the half step of a bfloat16 operand is allowed only where there is one:
bfloat16 rows aligned to 16 bytes.  Half precision, float32 and unaligned rows meet float32 operands, so their outputs are held to the
float32 sums and half a step of the result.  A subnormal power is off by 2^-150 at most, times a state's elements; that is below a step
of any bound here (2^-24 of the last token's own product)."""

import numpy as np
import pytest
import torch

from test_gpu_decay_attention import BF16, F16, F32, UNIT, call, make, oracle, tl, upload

pytestmark = pytest.mark.gpu

RATES = [0.0, -1e-4, -0.3, -2.7, -2.72, -2.74, -2.78, -2.9, -3.0, -3.2, -3.24, -3.26, -3.3, -8.0, -np.inf]


def check(c, out, state, rounded=None, in_place=False):
    """``rounded``: operands of the matrix instructions are rounded to bfloat16."""
    rounded = c.tag == BF16 if rounded is None else rounded
    want, size, want_state, bound = oracle(c, in_place)
    steps = (2 * max(int(c.q_lens.max()), 1) + 2 * c.Dk + 64) * 2.0 ** -24
    unit, halves, tiny = UNIT[c.tag], 2.0 ** -8 if rounded else 0.0, 2.0 ** -25 if c.tag == F16 else 0.0
    err = np.abs(tl.from_torch(out, c.tag) - want)
    assert (err <= unit * np.abs(want) + (1 + unit) * (steps + halves) * size + tiny).all()  # (NaN is not <=)
    assert (np.abs(state.cpu().numpy().astype(np.float64) - want_state) <= steps * bound).all()


@pytest.mark.parametrize("tag", [BF16, F32, F16])
@pytest.mark.parametrize("q_lens", [[64], [65, 1, 63], [150, 33, 97], [1500, 2, 130]])  # the last one is cut into segments
def test_every_decay(gpu, tag, q_lens):
    c = make(500 + len(q_lens), q_lens, Hq=len(RATES), Hkv=len(RATES), Dk=64, Dv=64, tag=tag, decays=np.array(RATES), past=[3] * len(q_lens))
    d = upload(c, gpu)
    out, state = call(d)
    torch.cuda.synchronize()
    check(c, out, state)


@pytest.mark.parametrize("tag", [BF16, F16])
def test_every_decay_with_shared_heads_in_place(gpu, tag):
    c = make(510, [130, 1, 64, 700], Hq=2 * len(RATES), Hkv=len(RATES), Dk=128, Dv=128, tag=tag, decays=np.array(RATES), past=[0, 4, 9, 1])
    d = upload(c, gpu)
    out, state = call(d, in_place=True)
    torch.cuda.synchronize()
    check(c, out, state, in_place=True)


def test_every_decay_of_unaligned_rows(gpu):
    c = make(520, [150, 900], Hq=len(RATES), Hkv=len(RATES), Dk=64, Dv=64, tag=BF16, decays=np.array(RATES))
    d = upload(c, gpu)
    for name in ("q", "k", "v"):
        x = d[name].flatten(1)
        d[name] = torch.cat([x[:, :1], x], dim=1)[:, 1:].unflatten(1, d[name].shape[1:])  # rows two bytes off
    out, state = call(d)
    torch.cuda.synchronize()
    check(c, out, state, rounded=False)


def test_random_batches_of_all_decays(gpu):
    for seed in range(18):
        rng = np.random.default_rng(7000 + seed)
        Hkv, n = int(rng.choice([1, 2, 3])), int(rng.integers(1, 6))
        lens = [int(x) for x in rng.choice([1, 2, 16, 17, 32, 64, 65, 96, 97, 200, 257, 400], size=n)]
        c = make(seed, lens, Hq=Hkv * int(rng.choice([1, 2, 4])), Hkv=Hkv, Dk=int(rng.choice([16, 64, 100, 128, 256])), Dv=int(rng.choice([16, 64, 72, 128, 256])),
                 tag=[F16, F32, BF16][seed % 3], past=rng.choice([0, 3], size=n), pad_rows=int(rng.integers(0, 3)), pad_tokens=int(rng.integers(0, 3)),
                 decays=rng.uniform(-8.0, -1e-4, Hkv))
        d = upload(c, gpu)
        out, state = call(d)
        torch.cuda.synchronize()
        # (bfloat16 rows of 100 keys or 72 values may take either kernel: the looser bound)
        check(c, out, state)
