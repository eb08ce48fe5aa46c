"""What the measurements of the append-with-rotation and decayed linear attention operators run.

Three operators of a serving step, each in the plain form (elementary torch operations in float32) and as the
calls a program makes of this package:

* ``append``: rotate the queries and keys of a ragged batch by their positions and write keys and values into the
  paged cache (interleaved K/V pages, separate pools, or scaled 8-bit pages);
* ``latent``: the same for the rope part of multi-latent attention and its latent pages;
* ``decay``: linear attention with one decay per KV head over a ragged batch, states in float32 slots.

A batch is described by plain numbers: ``decode`` rows of one token, ``prompts`` rows that share ``tokens`` tokens
unevenly (``shape`` seeds the split), ``past`` tokens at most in the cache before the call, ``pad`` token rows behind
the last sequence.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2, "fp8": 1, "int8": 1}
_QMAX = {"fp8": 448.0, "int8": 127.0}


def _append(name, **over):
    case = {"name": name, "op": "append", "layout": "pages", "heads": 32, "kv_heads": 8, "dim": 128, "stored": 128, "rope": 128,
            "neox": True, "src": "bf16", "kv": "bf16", "scaled": False, "page": 64, "decode": 0, "prompts": 0, "tokens": 0,
            "past": 0, "pad": 0, "fused": False, "shape": 1}
    return {**case, **over}


def _latent(name, **over):
    case = {"name": name, "op": "latent", "heads": 128, "rank": 512, "rope": 64, "neox": False, "src": "bf16", "kv": "bf16", "page": 64,
            "decode": 0, "prompts": 0, "tokens": 0, "past": 0, "pad": 0, "shape": 1}
    return {**case, **over}


def _decay(name, **over):
    case = {"name": name, "op": "decay", "heads": 32, "kv_heads": 32, "dk": 128, "dv": 128, "src": "bf16", "decode": 0, "prompts": 0,
            "tokens": 0, "past": 1, "pad": 0, "shape": 1}
    return {**case, **over}


def listed():
    return [
        # one user's next token, 32 query and 8 KV heads of 128: nothing but latency
        _append("append one token", decode=1, past=500),
        # the decode step of the benchmark's 256-sequence batch, q, k and v views of one fused projection
        _append("append decode 256", decode=256, past=500, fused=True),
        # four prompt chunks of about 2048 tokens, 64-token pages
        _append("append prompts 8192", prompts=4, tokens=8192, past=1000, fused=True),
        # 64 decode rows and four chunks over scaled fp8 pages, 40 query heads (the quantised decode shape's heads)
        _append("append fp8 mixed 2112", heads=40, kv="fp8", scaled=True, decode=64, prompts=4, tokens=2048, past=100),
        # separate K and V pools in half precision, head size 80 with half of it rotated, odd lengths
        _append("append pools odd", layout="pools", heads=12, kv_heads=4, dim=80, stored=80, rope=40, neox=False, src="f16", kv="f16",
                decode=7, prompts=5, tokens=1501, past=333, pad=3, page=32),
        # multi-latent decode: 128 heads, 512 + 64
        _latent("latent decode 256", decode=256, past=500),
        # multi-latent prompt chunks
        _latent("latent prompts 4096", prompts=3, tokens=4096, past=700),
        # recurrent form, eight users: the latency of a small decode step
        _decay("decay decode 8", decode=8),
        # recurrent form at a full batch: 256 states of 64 heads, 128 x 128
        _decay("decay decode 256", heads=64, kv_heads=64, decode=256),
        # one long prompt from a fresh state: chunks of one sequence in parallel
        _decay("decay prompt 16384", prompts=1, tokens=16384, past=0),
        # a mixed step: decode rows beside prompt chunks of uneven lengths
        _decay("decay mixed 8192", heads=64, kv_heads=64, decode=48, prompts=6, tokens=8144, past=2),
        # float32, two query heads to a state, keys narrower than values, odd lengths
        _decay("decay f32 odd", heads=16, kv_heads=8, dk=64, dv=96, src="f32", decode=3, prompts=4, tokens=2999, past=1, pad=5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rows(rng, decode, tokens):
    kind = rng.choice(("decode", "prompts", "both"))
    return {"decode": 0 if kind == "prompts" else _log(rng, 1, decode), "prompts": 0 if kind == "decode" else rng.randint(1, 7),
            "tokens": 0 if kind == "decode" else _log(rng, 7, tokens), "pad": rng.choice((0, 0, 1, 5)), "shape": rng.randint(1, 10 ** 6)}


def draw(rng):
    op = rng.choice(("append", "latent", "decay", "decay"))
    if op == "append":
        layout = rng.choice(("pages", "pages", "pools"))
        dim = rng.choice((64, 80, 96, 128, 128, 256))
        kv_heads = rng.choice((1, 2, 4, 8))
        src = rng.choice(("bf16", "bf16", "f16", "f32"))
        kv = rng.choice((src, src, "fp8")) if layout == "pages" else src
        scaled = kv == "fp8" and src != "f16" and rng.random() < 0.7
        if scaled and rng.random() < 0.3:
            kv = "int8"
        stored = -(-dim // 128) * 128 if layout == "pages" and dim != 64 else dim
        return {k: v for k, v in _append("", layout=layout, heads=kv_heads * rng.choice((1, 2, 5, 8)), kv_heads=kv_heads, dim=dim, stored=stored,
                                         rope=rng.choice((dim, dim, dim // 2, dim // 4)), neox=rng.random() < 0.6, src=src, kv=kv, scaled=scaled,
                                         page=rng.choice((16, 32, 64, 128)), past=rng.randint(0, 900), fused=rng.random() < 0.4,
                                         **_rows(rng, 300, 6000)).items() if k != "name"}
    if op == "latent":
        src = rng.choice(("bf16", "bf16", "f16", "f32"))
        return {k: v for k, v in _latent("", heads=rng.choice((8, 16, 40, 128)), rank=rng.choice((512, 512, 256, 64)), rope=rng.choice((64, 64, 32, 128)),
                                         neox=rng.random() < 0.4, src=src, kv=rng.choice((src, src, "fp8")), page=rng.choice((16, 32, 64)),
                                         past=rng.randint(0, 900), **_rows(rng, 300, 4000)).items() if k != "name"}
    kv_heads = rng.choice((2, 4, 8, 16, 32))
    return {k: v for k, v in _decay("", heads=kv_heads * rng.choice((1, 1, 1, 2, 4)), kv_heads=kv_heads, dk=rng.choice((32, 64, 80, 128, 128, 256)),
                                    dv=rng.choice((64, 96, 128, 128, 200)), src=rng.choice(("bf16", "bf16", "bf16", "f16", "f32")),
                                    past=rng.choice((0, 1, 2)), **_rows(rng, 100, 6000)).items() if k != "name"}


# ---- the batch that a case's numbers describe -----------------------------------------------------------


def _lengths(case):
    """New tokens of each sequence and the tokens before them, decode rows and prompts in a shuffled order."""
    r = random.Random(case["shape"])
    lens = [1] * case["decode"]
    if case["prompts"]:
        n, left = case["prompts"], case["tokens"] - case["prompts"]
        weight = [r.uniform(0.3, 1.0) for _ in range(n)]
        share = [int(left * w / sum(weight)) for w in weight]
        share[0] += left - sum(share)
        lens += [1 + s for s in share]
    r.shuffle(lens)
    if case["op"] == "decay":  # past: 0 every sequence is fresh, 1 every one goes on, 2 some of both
        past = [0 if case["past"] == 0 or (case["past"] == 2 and r.random() < 0.5) else 100 for _ in lens]
    else:
        past = [r.randint(0, case["past"]) for _ in lens]
    return lens, past


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _batch(case):
    lens, past = _lengths(case)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    return {"case": case, "lens": lens, "past": past, "tokens": starts[-1], "rows": starts[-1] + case["pad"], "starts": starts,
            "query_start_loc": _ints(starts), "context_lens": _ints([n + p for n, p in zip(lens, past)]), "num_seqs": _ints([len(lens)])}


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _table(positions, dim):
    """cos | sin of the rotation's angles, base 10000, computed in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), dim=1).float().contiguous()


def _tables(case, s, gen):
    pages = [-(-(n + p) // case["page"]) for n, p in zip(s["lens"], s["past"])]
    order = (torch.randperm(sum(pages), generator=gen, device="cuda") + 1).tolist()  # page 0 is nobody's
    rows, at, width = [], 0, max(pages)
    for n in pages:
        rows.append(order[at:at + n] + [0] * (width - n))
        at += n
    s["block_tables"] = _ints(rows)
    return sum(pages) + 1


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s = _batch(case)
    T, src = s["rows"], _TYPES[case["src"]]
    if case["op"] == "decay":
        H, K, dk, dv, n = case["heads"], case["kv_heads"], case["dk"], case["dv"], len(s["lens"])
        s["query"], s["key"], s["value"] = (_normal(gen, sh, src) for sh in ((T, H, dk), (T, K, dk), (T, K, dv)))
        low, high = math.log(1e-3), math.log(1.0)
        s["log_decay"] = -torch.exp(torch.rand(K, generator=gen, device="cuda") * (high - low) + low)
        # every sequence reads its state from one slot and leaves the new one in another, as where prefixes are kept
        s["state"] = _normal(gen, (2 * n, K, dk, dv), torch.float32)
        slots = torch.randperm(2 * n, generator=gen, device="cuda").to(torch.int32)
        s["state_indices"], s["state_out_indices"] = slots[:n].contiguous(), slots[n:].contiguous()
        chunk = min(64, max(s["lens"]))
        cut = [(i, at, min(chunk, m - at)) for i, m in enumerate(s["lens"]) for at in range(0, m, chunk)]
        s["chunk"] = chunk
        s["cut"] = _ints([[i, at, m, s["starts"][i] + at] for i, at, m in cut])
        s["last"] = _ints([max(j for j, c in enumerate(cut) if c[0] == i) for i in range(n)]).long()
        return s
    P = _tables(case, s, gen)
    s["cos_sin"] = _table(max(n + p for n, p in zip(s["lens"], s["past"])), case["rope"])
    kv = _TYPES[case["kv"]]
    if case["op"] == "latent":
        s["queries_pe"] = _normal(gen, (T, case["heads"], case["rope"]), src)
        s["keys_values"] = _normal(gen, (T, case["rank"]), src).to(kv)
        s["keys_pe"] = _normal(gen, (T, case["rope"]), src)
        width = -(-case["rank"] // 128) * 128 + -(-case["rope"] // 128) * 128
        s["kv_pages"] = _normal(gen, (P, case["page"], width), torch.float32).to(kv)
        return s
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    if case["fused"]:  # views of one projection's output
        qkv = _normal(gen, (T, (H + 2 * K) * D), src)
        s["query"], s["key"], s["value"] = (x.unflatten(1, (-1, D)) for x in qkv.split((H * D, K * D, K * D), dim=1))
    else:
        s["query"], s["key"], s["value"] = (_normal(gen, (T, h, D), src) for h in (H, K, K))
    if case["layout"] == "pools":
        s["key_cache"], s["value_cache"] = (_normal(gen, (P, case["page"], K, D), kv) for _ in range(2))
        return s
    pages = torch.randn((P, case["page"], 2 * K, case["stored"]), generator=gen, device="cuda")
    pages[..., D:] = 0
    if case["scaled"]:
        pages = pages * (_QMAX[case["kv"]] / 5)
        pages = pages.round().clamp(-127, 127) if case["kv"] == "int8" else pages.clamp(-448, 448)
        s["kv_scales"] = torch.rand((P, 2 * K), generator=gen, device="cuda") * 0.005 + 0.007
    s["kv_pages"] = pages.to(kv)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------


def _places(s, page):
    """Sequence, position and (page, slot) of every token."""
    at = torch.arange(s["tokens"], device="cuda")
    qsl = s["query_start_loc"].long()
    seq = (at[:, None] >= qsl[None, 1:]).sum(1)
    end = qsl[1:][seq]
    position = s["context_lens"].long()[seq] - end + at
    return position, s["block_tables"].long()[seq, position // page], position % page


def _rotate(x, angles, rope, neox):
    x = x.float()
    half = rope // 2
    c, n = angles[:, None, :half], angles[:, None, half:]
    a, b = (x[..., :half], x[..., half:rope]) if neox else (x[..., 0:rope:2], x[..., 1:rope:2])
    first, second = a * c - b * n, b * c + a * n
    turned = torch.cat((first, second), dim=-1) if neox else torch.stack((first, second), dim=-1).flatten(-2)
    return torch.cat((turned, x[..., rope:]), dim=-1)


def _behind(x, rows):
    """Rows of zeros behind the last sequence."""
    return torch.cat((x, x.new_zeros((rows - x.shape[0], *x.shape[1:])))) if rows > x.shape[0] else x


def _coded(x, kv):
    q = _QMAX[kv]
    x = x.clamp(-q, q)
    return x.round() if kv == "int8" else x.to(torch.float8_e4m3fn).to(x.dtype)


def _append_scaled(s, new, page, slot):
    """New float values into scaled 8-bit pages: a page's scale only grows, and what it held is coded again."""
    case, pages, scales = s["case"], s["kv_pages"], s["kv_scales"]
    D, slots = case["dim"], torch.arange(case["page"], device="cuda")
    most = torch.zeros_like(scales).index_reduce_(0, page, new.abs().amax(-1), "amax")
    first = torch.full((pages.shape[0],), case["page"], device="cuda").index_reduce_(0, page, slot, "amin")
    touched = first < case["page"]
    old = torch.where((first == 0)[:, None], torch.zeros_like(scales), scales)
    grown = torch.maximum(old, most / _QMAX[case["kv"]])
    grown = torch.where(touched[:, None], torch.where(grown == 0, torch.ones_like(grown), grown), scales)
    held = pages.to(new.dtype)
    again = _coded(held[..., :D] * old[:, None, :, None] / grown[:, None, :, None], case["kv"])
    redo = (touched[:, None] & (slots[None] < first[:, None]))[..., None] & (grown > old)[:, None]
    held[..., :D] = torch.where(redo[..., None], again, held[..., :D])
    coded = _coded(new / grown[page][..., None], case["kv"])
    held[page, slot] = torch.cat((coded, coded.new_zeros((*coded.shape[:2], pages.shape[-1] - D))), dim=-1)
    return held, grown


def _plain_append(s):
    case = s["case"]
    n, src = s["tokens"], _TYPES[case["src"]]
    position, page, slot = _places(s, case["page"])
    angles = s["cos_sin"][position]
    query = _behind(_rotate(s["query"][:n], angles, case["rope"], case["neox"]).to(src), s["rows"])
    key, value = _rotate(s["key"][:n], angles, case["rope"], case["neox"]), s["value"][:n].float()
    if case["layout"] == "pools":
        s["key_cache"][page, slot] = key.to(s["key_cache"].dtype)
        s["value_cache"][page, slot] = value.to(s["value_cache"].dtype)
        return query, s["key_cache"], s["value_cache"]
    new = torch.stack((key, value), dim=2).flatten(1, 2)
    if case["scaled"]:
        held, grown = _append_scaled(s, new, page, slot)
        s["kv_pages"].copy_(held)
        s["kv_scales"].copy_(grown)
        return query, _values(s), s["kv_scales"]
    new = torch.cat((new, new.new_zeros((*new.shape[:2], case["stored"] - case["dim"]))), dim=-1)
    _put(s["kv_pages"], page, slot, new.to(s["kv_pages"].dtype))
    return query, s["kv_pages"]


def _put(pages, page, slot, rows):
    """rows into their places; 8-bit floats as bytes, for which torch has no indexed store."""
    if pages.dtype == torch.float8_e4m3fn:
        pages, rows = pages.view(torch.uint8), rows.view(torch.uint8)
    pages[page, slot] = rows


def _values(s):
    """What the scaled codes stand for."""
    return s["kv_pages"].float() * s["kv_scales"][:, None, :, None]


def _plain_latent(s):
    case = s["case"]
    n, rank, rope = s["tokens"], case["rank"], case["rope"]
    position, page, slot = _places(s, case["page"])
    angles = s["cos_sin"][position]
    queries = _behind(_rotate(s["queries_pe"][:n], angles, rope, case["neox"]).to(_TYPES[case["src"]]), s["rows"])
    turned = _rotate(s["keys_pe"][:n, None], angles, rope, case["neox"])[:, 0].to(s["kv_pages"].dtype)
    row = torch.zeros((n, s["kv_pages"].shape[-1]), device="cuda").to(s["kv_pages"].dtype)
    at = -(-rank // 128) * 128
    row[:, :rank] = s["keys_values"][:n]
    row[:, at:at + rope] = turned
    _put(s["kv_pages"], page, slot, row)
    return queries, s["kv_pages"]


def _plain_decay(s):
    """Chunks of up to 64 tokens: inside a chunk by the masked product of queries and keys, across chunks by states."""
    case = s["case"]
    H, K, dk, dv, C = case["heads"], case["kv_heads"], case["dk"], case["dv"], s["chunk"]
    seq, at, size, start = s["cut"].long().unbind(1)
    N, n, G = seq.shape[0], len(s["lens"]), H // K
    g = s["log_decay"].float()
    step = torch.arange(C, device="cuda")
    here = step[None] < size[:, None]
    rows = torch.where(here, start[:, None] + step, torch.zeros_like(step))
    q, k, v = (torch.where(here[..., None, None], s[name].float()[rows], 0.0).transpose(1, 2) for name in ("query", "key", "value"))
    past = s["context_lens"].long() > (s["query_start_loc"][1:] - s["query_start_loc"][:-1]).long()
    first = torch.where(past[:, None, None, None], s["state"][s["state_indices"].long()], 0.0)  # [n, K, dk, dv]
    # what each chunk adds to its state: sum over its tokens, each decayed to the chunk's end
    left = (size[:, None] - 1 - step).clamp(min=0)
    weight = torch.exp(g[None, :, None] * left[:, None])
    local = torch.matmul((k * weight[..., None]).transpose(-1, -2).contiguous(), v)  # [N, K, dk, dv]
    begin = first[seq] * torch.exp(g[None] * at[:, None])[..., None, None]
    if N > n:  # the chunks of one sequence before this one, decayed over the tokens between
        gap = at[:, None] - at[None] - size[None]
        before = (seq[:, None] == seq[None]) & (gap >= 0)
        carry = torch.where(before[None], torch.exp(g[:, None, None] * gap.clamp(min=0)), 0.0)
        begin = begin + torch.matmul(carry, local.transpose(0, 1).reshape(K, N, dk * dv)).reshape(K, N, dk, dv).transpose(0, 1)
    q = q.unflatten(1, (K, G))  # [N, K, G, C, dk]
    gap = step[:, None] - step[None]
    within = torch.where(gap >= 0, torch.exp(g[:, None, None] * gap.clamp(min=0)), 0.0)
    scores = torch.matmul(q, k[:, :, None].transpose(-1, -2).contiguous()) * within[:, None]
    out = torch.matmul(scores, v[:, :, None])
    out = out + torch.matmul(q * torch.exp(g[:, None] * (step + 1))[:, None, :, None], begin[:, :, None])
    out = (out * dk ** -0.5).flatten(1, 2).transpose(1, 2)  # [N, C, H, dv]
    result = torch.zeros((s["rows"] + 1, H, dv), device="cuda")
    result[torch.where(here, rows, s["rows"])] = out  # places behind a chunk's end go to a row that is dropped
    end = begin * torch.exp(g[None] * size[:, None])[..., None, None] + local
    s["state"][s["state_out_indices"].long()] = end[s["last"]]
    return result[:-1].to(_TYPES[case["src"]]), s["state"]


# ---- the package's calls --------------------------------------------------------------------------------


def _own_append(s):
    from easydel_amd import kernels

    case = s["case"]
    if case["layout"] == "pools":
        return kernels.rope_unified_page_scatter(s["query"], s["key"], s["value"], s["key_cache"], s["value_cache"], s["cos_sin"],
                                                 s["context_lens"], s["block_tables"], s["query_start_loc"], s["num_seqs"],
                                                 is_neox_style=case["neox"])
    done = kernels.rope_page_scatter_ragged(s["query"], s["key"], s["value"], s["kv_pages"], s["cos_sin"], s["context_lens"],
                                            s["block_tables"], s["query_start_loc"], s["num_seqs"], is_neox_style=case["neox"],
                                            kv_scales=s["kv_scales"] if case["scaled"] else None)
    return (done[0], _values(s), done[2]) if case["scaled"] else done


def _own_latent(s):
    from easydel_amd import kernels

    return kernels.rope_mla_page_scatter(s["queries_pe"], s["keys_values"], s["keys_pe"], s["kv_pages"], s["cos_sin"], s["context_lens"],
                                         s["block_tables"], s["query_start_loc"], s["num_seqs"], is_neox_style=s["case"]["neox"])


def _own_decay(s):
    from easydel_amd import kernels

    return kernels.decay_linear_attention(s["query"], s["key"], s["value"], s["log_decay"], s["state"], s["state_indices"],
                                          s["query_start_loc"], s["num_seqs"], context_lens=s["context_lens"],
                                          state_out_indices=s["state_out_indices"])


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_append(state) if op == "append" else _own_latent(state) if op == "latent" else _own_decay(state)
    return _plain_append(state) if op == "append" else _plain_latent(state) if op == "latent" else _plain_decay(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------


def work(case):
    lens, past = _lengths(case)
    n, e = sum(lens), _BYTES[case["src"]]
    if case["op"] == "decay":
        H, K, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
        states = (len(lens) + sum(p > 0 for p in past)) * K * dk * dv * 4
        return {"bytes": n * (H * (dk + dv) + K * (dk + dv)) * e + states, "flops": n * 2 * dk * dv * (H + K)}
    angles = n * case["rope"] * 4
    if case["op"] == "latent":
        width = -(-case["rank"] // 128) * 128 + -(-case["rope"] // 128) * 128
        kv = _BYTES[case["kv"]]
        return {"bytes": n * (2 * case["heads"] * case["rope"] * e + case["rope"] * e + (case["rank"] + width) * kv) + angles,
                "flops": 3 * n * (case["heads"] + 1) * case["rope"]}
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    moved = n * ((2 * H + 2 * K) * D * e + 2 * K * case["stored"] * _BYTES[case["kv"]])
    if case["scaled"]:  # what run returns are the values that the codes stand for: the whole pool's
        pool = (sum(-(-(m + p) // case["page"]) for m, p in zip(lens, past)) + 1) * case["page"] * 2 * K * case["stored"]
        moved += pool * 5
    return {"bytes": moved + angles, "flops": 3 * n * (H + K) * case["rope"]}


# ---- the definitions in 64 bits, token by token ---------------------------------------------------------


def _turned(x, angle, rope, neox):
    """x [.., D] at one angle row each, as complex numbers."""
    x = x.double()
    half = rope // 2
    unit = torch.complex(angle[:, :half].double(), angle[:, half:].double())[:, None]
    pairs = torch.stack((x[..., :half], x[..., half:rope]), -1) if neox else x[..., :rope].unflatten(-1, (half, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
    y = x.clone()
    y[..., :rope] = torch.cat((z[..., 0], z[..., 1]), -1) if neox else z.flatten(-2)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_decay(s) if case["op"] == "decay" else _exact_written(s)


def _exact_written(s):
    case, n = s["case"], s["tokens"]
    table = s["block_tables"].tolist()
    where = [(i, p + r) for i, (m, p) in enumerate(zip(s["lens"], s["past"])) for r in range(m)]
    position = torch.tensor([w for _, w in where], device="cuda")
    page = torch.tensor([table[i][w // case["page"]] for i, w in where], device="cuda")
    slot, angle = position % case["page"], s["cos_sin"][position]
    rope, neox = case["rope"], case["neox"]
    asked = s["queries_pe" if case["op"] == "latent" else "query"]
    query = torch.zeros(asked.shape, dtype=torch.float64, device="cuda")
    query[:n] = _turned(asked[:n], angle, rope, neox)
    if case["op"] == "latent":
        pages, at = s["kv_pages"].double(), -(-case["rank"] // 128) * 128
        pages[page, slot] = 0.0
        pages[page, slot, :case["rank"]] = s["keys_values"][:n].double()
        pages[page, slot, at:at + rope] = _turned(s["keys_pe"][:n, None], angle, rope, neox)[:, 0]
        return query, pages
    key, value = _turned(s["key"][:n], angle, rope, neox), s["value"][:n].double()
    if case["layout"] == "pools":
        pools = [s["key_cache"].double(), s["value_cache"].double()]
        pools[0][page, slot], pools[1][page, slot] = key, value
        return query, *pools
    pages, D = s["kv_pages"].double(), case["dim"]
    if not case["scaled"]:
        pages[page, slot] = 0.0
        pages[page, slot, 0::2, :D], pages[page, slot, 1::2, :D] = key, value
        return query, pages
    scales, qmax = s["kv_scales"].double(), _QMAX[case["kv"]]
    fresh = torch.zeros_like(pages)
    fresh[page, slot, 0::2, :D], fresh[page, slot, 1::2, :D] = key, value
    new = torch.zeros(pages.shape[:2], dtype=torch.bool, device="cuda")
    new[page, slot] = True
    touched, begun = new.any(1), new[:, 0]
    old = scales * (~begun[:, None]).double()
    grown = torch.maximum(old, fresh.abs().amax((1, 3)) / qmax)
    grown[grown == 0] = 1.0
    grown = torch.where(touched[:, None], grown, scales)
    unit = grown[:, None, :, None]
    kept = torch.cumsum(new.int(), 1) == 0  # slots in front of a page's first new token
    redo = (touched[:, None] & kept)[:, :, None, None] & (grown > old)[:, None, :, None]
    pages = torch.where(redo, _coded(pages * old[:, None, :, None] / unit, case["kv"]), pages)
    pages = torch.where(new[:, :, None, None], _coded(fresh / unit, case["kv"]), pages)
    return query, pages * unit, grown


def _exact_decay(s):
    """The recurrence itself, all sequences a token at a time, the longest first so that the ended ones drop out."""
    case, n = s["case"], len(s["lens"])
    G = case["heads"] // case["kv_heads"]
    longest = max(s["lens"])
    if longest > 40000:
        return None
    order = sorted(range(n), key=lambda i: -s["lens"][i])
    lens = [s["lens"][i] for i in order]
    idx = torch.tensor(order, device="cuda")
    start = torch.tensor([s["starts"][i] for i in order], device="cuda")
    fresh = torch.tensor([s["past"][i] == 0 for i in order], device="cuda")
    state = s["state"].double()
    S = state[s["state_indices"].long()[idx]]
    S[fresh] = 0.0
    decay = torch.exp(s["log_decay"].double())[None, :, None, None]
    out = torch.zeros((s["rows"], case["heads"], case["dv"]), dtype=torch.float64, device="cuda")
    live = n
    for t in range(longest):
        while lens[live - 1] <= t:
            live -= 1
        row = start[:live] + t
        q, k, v = (s[name][row].double() for name in ("query", "key", "value"))
        now = S[:live]
        now *= decay
        now += k[..., :, None] * v[..., None, :]
        out[row] = (torch.matmul(q.unflatten(1, (-1, G)), now) * case["dk"] ** -0.5).flatten(1, 2)
    state[s["state_out_indices"].long()[idx]] = S
    return out, state
