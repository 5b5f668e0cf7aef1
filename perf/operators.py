"""The quantized K/V cache operators as measured cases.

Three calls of ``QuantKVCache`` are measured, in two kinds of case:

* ``store``   ``write`` quantizes the K/V rows of a call into the cache and
              ``read`` reads the same rows back; the outputs are the values
              the cache now stands for.
* ``attend``  ``attend``: causal attention of a call's query rows over the
              quantized rows of their sequences.

A call's rows come in segments: segment b holds ``count`` rows at positions
``start .. start + count - 1`` of sequence b; query row i of a segment
attends to positions ``0 .. start + i``.

The stored format: head_dim is cut into groups of 32 values; with a the
group's largest magnitude and L = 7 (4 bits) or 127 (8 bits) the group holds
the scale s = bf16(a / L) and the codes c = clamp(rint(x / s), -L, L) (0 where
s is 0), and stands for s * c.
"""

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_GROUP = 32


# ------------------------------------------------------------------- cases
def _attend(name, **kw):
    case = dict(name=name, kind="attend", dtype="bf16", bits=4, q_heads=16, kv_heads=8, head_dim=128, seqs=1, low=0,
                high=0, rows_low=1, rows_high=1, mix=1)
    case.update(kw)
    return case


def _store(name, **kw):
    case = dict(name=name, kind="store", dtype="bf16", bits=4, q_heads=0, kv_heads=8, head_dim=128, seqs=1, low=0,
                high=0, rows_low=1, rows_high=1, mix=1)
    case.update(kw)
    return case


def listed():
    return [
        # a single stream just after a 16-token prompt: nothing but latency
        _attend("attend-1x17", low=16, high=16),
        # a single stream at about 1k tokens, the decode benchmark's context;
        # fp32 queries, as the layers' activations are
        _attend("attend-1x1k-fp32", dtype="fp32", low=1279, high=1279),
        # one stream over a long document
        _attend("attend-1x32k", low=32767, high=32767),
        # the batch-64 decode step after 1024-token prompts
        _attend("attend-64x1k", seqs=64, low=1024, high=1279),
        # a full batch of 8k contexts: the K/V bytes are all that counts
        _attend("attend-64x8k", seqs=64, low=8100, high=8191),
        # a serving mix: lengths from one token to 20k, four query heads a
        # K/V head, fp16, the cache in 8 bits
        _attend("attend-ragged-8bit", dtype="fp16", bits=8, q_heads=32, seqs=24, low=0, high=20000, mix=5),
        # checking a few proposed tokens a sequence in one pass; 64-wide heads
        _attend("attend-check-5", q_heads=12, kv_heads=3, head_dim=64, seqs=16, low=1000, high=5000, rows_low=3,
                rows_high=5, mix=6),
        # a fresh 1024-token prompt
        _attend("attend-prompt-1k", rows_low=1024, rows_high=1024),
        # the last 1000-odd tokens of an 8k prompt that is fed in chunks
        _attend("attend-chunk-8k", low=7169, high=7169, rows_low=1023, rows_high=1023),
        # one decode step's rows of four sequences
        _store("store-step-4", seqs=4, low=1024, high=1100),
        # ragged prompts of fp32 rows into an 8-bit cache of 64-wide heads
        _store("store-ragged-8bit", dtype="fp32", bits=8, kv_heads=6, head_dim=64, seqs=7, low=0, high=300, rows_low=1,
               rows_high=1500, mix=3),
        # prompts of a whole batch
        _store("store-prompts", seqs=16, rows_low=2000, rows_high=2048, mix=2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    head_dim = rng.choice([64, 128, 128])
    kv_heads = rng.randint(1, 8)
    case = dict(dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), bits=rng.choice([4, 4, 8]), head_dim=head_dim,
                kv_heads=kv_heads, q_heads=kv_heads * rng.choice([1, 2, 2, 4, 8]), mix=rng.randint(0, 10**6))
    what = rng.choice(["decode", "decode", "chunk", "store"])
    if what == "store":
        case.update(kind="store", q_heads=0, seqs=_log(rng, 1, 16), low=0, high=rng.randint(0, 700))
        case["rows_high"] = _log(rng, 1, 2048)
        case["rows_low"] = rng.randint(1, case["rows_high"])
        if case["dtype"] == "fp32":  # no dearer than the largest listed case
            case["seqs"] = min(case["seqs"], 8)
        return case
    case["kind"] = "attend"
    if what == "decode":
        case["seqs"] = _log(rng, 1, 64)
        case["high"] = _log(rng, 1, min(32767, 8191 * 64 // case["seqs"]) // (2 if case["bits"] == 8 else 1))
        case["low"] = rng.randint(0, case["high"])
        case["rows_low"] = case["rows_high"] = 1
        return case
    case["q_heads"] = min(case["q_heads"], 16)
    case["q_heads"] -= case["q_heads"] % kv_heads
    case["rows_high"] = _log(rng, 2, 1023)
    case["rows_low"] = rng.randint(1, case["rows_high"])
    room = 1023 * 7000 // case["rows_high"]  # sequences x positions, no dearer than the largest listed case
    case["seqs"] = _log(rng, 1, 8)
    case["high"] = _log(rng, 1, max(1, min(30000, room // case["seqs"] - case["rows_high"])))
    case["low"] = rng.randint(0, case["high"])
    return case


def _segments(case):
    """(start, count) of each sequence, from the case alone."""
    rng = random.Random(case["mix"])
    out = []
    for _ in range(case["seqs"]):
        start = rng.randint(case["low"], case["high"])
        out.append((start, rng.randint(case["rows_low"], case["rows_high"])))
    return out


def work(case):
    segs = _segments(case)
    d, hk, hq = case["head_dim"], case["kv_heads"], case["q_heads"]
    size = torch.empty(0, dtype=_TYPES[case["dtype"]]).element_size()
    row = 2 * hk * (d * case["bits"] // 8 + d // _GROUP * 2)  # K and V of one position: codes and scales
    rows = sum(c for _, c in segs)
    if case["kind"] == "store":
        # rows in, codes and scales written and read, values out; scaling and rounding of each value, its product
        return {"bytes": rows * (2 * 2 * hk * d * size + 2 * row), "flops": rows * 2 * hk * d * 3}
    seen = sum(s + c for s, c in segs)
    pairs = sum(c * s + c * (c + 1) // 2 for s, c in segs)
    return {"bytes": seen * row + 2 * rows * hq * d * size, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------- inputs
def _kv(case, gen, rows):
    """K and V rows of one sequence, [rows, kv_heads, head_dim]: K with
    channels of unlike spread, as after a weighted norm."""
    shape = (rows, case["kv_heads"], case["head_dim"])
    t = _TYPES[case["dtype"]]
    gain = torch.exp(0.4 * torch.randn(shape[1:], generator=gen, device="cuda"))
    k = (torch.randn(shape, generator=gen, device="cuda") * gain).to(t)
    v = (torch.randn(shape, generator=gen, device="cuda") * 0.7).to(t)
    return k, v


def _inputs(case, seed):
    """Per sequence the K/V rows (a store: the call's rows; an attend: every
    position up to the segment's end), and the query rows of an attend."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    segs = _segments(case)
    kv = [_kv(case, gen, c if case["kind"] == "store" else s + c) for s, c in segs]
    q = None
    if case["kind"] == "attend":
        rows = sum(c for _, c in segs)
        q = 1.5 * torch.randn(rows, case["q_heads"], case["head_dim"], generator=gen, device="cuda")
        q = q.to(_TYPES[case["dtype"]])
    return segs, kv, q


# --------------------------------------------------------------- plain form
def _quantize(x, bits):
    """Codes (int8) and scales (bf16) of rows x [..., head_dim]; the division
    in 64 bits, so that values next to a rounding border fall on its right
    side."""
    top = 7 if bits == 4 else 127
    g = x.double().unflatten(-1, (-1, _GROUP))
    scale = (g.abs().amax(-1) / top).to(torch.bfloat16)
    s = scale.double().unsqueeze(-1)
    code = torch.where(s > 0, (g / torch.where(s > 0, s, 1.0)).round().clamp(-top, top), 0.0)
    return code.to(torch.int8), scale


def _values(code, scale):
    """fp32 values of codes [..., groups, 32] and scales [..., groups]."""
    return (code.float() * scale.float().unsqueeze(-1)).flatten(-2)


def _plain_attend(case, segs, cache, q):
    out, r = [], 0
    hk, d = case["kv_heads"], case["head_dim"]
    ratio = case["q_heads"] // hk
    for (start, count), (kc, ks, vc, vs) in zip(segs, cache):
        k = _values(kc, ks).transpose(0, 1)  # [hk, positions, d]
        v = _values(vc, vs).transpose(0, 1)
        x = q[r:r + count].float().view(count, hk, ratio, d).permute(1, 2, 0, 3).reshape(hk, ratio * count, d)
        score = (x @ k.transpose(1, 2)) * (1.0 / math.sqrt(d))
        pos = torch.arange(start + count, device=q.device)
        own_pos = (start + torch.arange(count, device=q.device)).repeat(ratio)
        score = torch.where(pos[None, None, :] <= own_pos[None, :, None], score, -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        o = (p @ v) / p.sum(-1, keepdim=True)
        out.append(o.view(hk, ratio, count, d).permute(2, 0, 1, 3).reshape(count, hk * ratio, d))
        r += count
    return torch.cat(out).to(q.dtype)


# ------------------------------------------------------------ the interface
def prepare(case, seed):
    segs, kv, q = _inputs(case, seed)
    state = {"case": case, "segs": segs}
    store = case["kind"] == "store"
    if own:
        from qwen_megakernel_b200 import KVRows, QuantKVCache

        state["cache"] = QuantKVCache(case["seqs"], max(s + c for s, c in segs), num_kv_heads=case["kv_heads"],
                                      head_dim=case["head_dim"], bits=case["bits"], device="cuda")
        state["rows"] = KVRows([s for s, _ in segs], [c for _, c in segs], device="cuda")
        if not store:
            for b, (k, v) in enumerate(kv):
                state["cache"].write(k, v, KVRows([0], [len(k)], [b], device="cuda"))
    elif not store:
        state["cache"] = [_quantize(k, case["bits"]) + _quantize(v, case["bits"]) for k, v in kv]
    if store:
        state["k"] = torch.cat([k for k, _ in kv])
        state["v"] = torch.cat([v for _, v in kv])
    else:
        state["q"] = q
    return state


def run(state):
    case = state["case"]
    if case["kind"] == "store":
        t = _TYPES[case["dtype"]]
        if own:
            state["cache"].write(state["k"], state["v"], state["rows"])
            k, v = state["cache"].read(state["rows"], dtype=t)
        else:
            k = _values(*_quantize(state["k"], case["bits"])).to(t)
            v = _values(*_quantize(state["v"], case["bits"])).to(t)
        return {"k": k, "v": v}
    if own:
        return state["cache"].attend(state["q"], state["rows"])
    return _plain_attend(case, state["segs"], state["cache"], state["q"])


def exact(case, seed):
    """What run returns, in 64 bits from the definition."""
    segs, kv, q = _inputs(case, seed)
    top = 2 ** (case["bits"] - 1) - 1

    def held(x):  # the values a cache row stands for
        y = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        for g in range(0, x.shape[-1], _GROUP):
            part = x[..., g:g + _GROUP].double()
            s = (part.abs().max(dim=-1, keepdim=True).values / top).bfloat16().double()
            y[..., g:g + _GROUP] = s * torch.nan_to_num(part / s).round().clamp(-top, top)
        return y

    if case["kind"] == "store":
        return {"k": torch.cat([held(k) for k, _ in kv]), "v": torch.cat([held(v) for _, v in kv])}
    ratio = case["q_heads"] // case["kv_heads"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    r = 0
    for (start, count), (k, v) in zip(segs, kv):
        k, v = held(k), held(v)
        live = torch.ones(count, start + count, dtype=torch.bool, device=q.device).tril(start)
        for h in range(case["q_heads"]):
            score = q[r:r + count, h].double() @ k[:, h // ratio].T / math.sqrt(case["head_dim"])
            p = torch.softmax(score.masked_fill(~live, -math.inf), dim=-1)
            out[r:r + count, h] = p @ v[:, h // ratio]
        r += count
    return out
