"""Operators of generation over a 4-bit cache and of beam search, as cases that can be timed and compared.

Four operators, each in a plain form (elementary torch operations) and through the framework's entry points:

* ``store``: rows of keys and values are quantised into a cache of 4 bits at their sequences' positions, and the same positions
  are read back (``Cache4.append``, ``Cache4.read``);
* ``attend``: queries of one token, of a portion or of a whole prompt over that cache (``Cache4.attend``);
* ``select``: the best continuations over a sequence's beams and the vocabulary (``ops.beam_select``);
* ``reorder``: the beams' states follow the beams they continue (``ops.reorder_states``).

A cache row is held in groups of 32 columns: the smallest value m and the step s = (largest - smallest) / 15, each rounded to
float16, and per column the nearest code of 0 .. 15 to (x - m) / s; the code stands for m + s code.

Everything is made on the GPU from the case and a seed.  ``exact`` restates each operator in float64; it shares no code with the
plain forms.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rotor-rag_b200"))

own = False

GROUP = 32
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # a generation step of one sequence of the 2B model: one row of five heads, as float32 as its projections leave it
        dict(name="store_one", kind="store", batch=1, seq=1, kv=5, dim=128, past=1024, room=2048, dtype="float32", stacked=False),
        # a batch of prompts; keys and values are columns of the stacked q/k/v rows a product left
        dict(name="store_prompt", kind="store", batch=8, seq=2048, kv=5, dim=128, past=0, room=2304, dtype="bfloat16", stacked=True),
        # a portion behind cached rows, sizes that are multiples of nothing, heads of 64
        dict(name="store_ragged", kind="store", batch=3, seq=333, kv=7, dim=64, past=517, room=1111, dtype="float16", stacked=False),
        # one token of one sequence behind a prompt, as in the 2B model's generation: latency
        dict(name="attend_one", kind="attend", batch=1, seq=1, heads=20, kv=5, dim=128, low=1024, high=1024, window=0, sinks=False,
             dtype="float32"),
        # a step of 64 sequences of the larger shape, cached lengths between one and four thousand: the serving load
        dict(name="attend_batch", kind="attend", batch=64, seq=1, heads=64, kv=8, dim=128, low=1024, high=4095, window=0, sinks=False,
             dtype="bfloat16"),
        # one sequence with a long document behind it
        dict(name="attend_long", kind="attend", batch=1, seq=1, heads=64, kv=8, dim=128, low=131000, high=131000, window=0, sinks=False,
             dtype="float16"),
        # a few tokens behind a window, heads of 64 with sinks, float32 in and out
        dict(name="attend_portion", kind="attend", batch=3, seq=9, heads=12, kv=4, dim=64, low=700, high=1900, window=777, sinks=True,
             dtype="float32"),
        # prompts over their own freshly written rows
        dict(name="attend_prompt", kind="attend", batch=8, seq=2048, heads=20, kv=5, dim=128, low=0, high=0, window=0, sinks=False,
             dtype="bfloat16"),
        # beams of one request, twice as many candidates as beams so that ended ones can be set aside
        dict(name="select_few", kind="select", groups=1, width=4, vocab=102400, count=8, ended=0, dtype="float32"),
        # beams of a batch of requests over the largest vocabulary, some of them ended
        dict(name="select_many", kind="select", groups=16, width=8, vocab=128256, count=16, ended=2, dtype="float32"),
        # the 4-bit cache of one layer behind one request's beams
        dict(name="reorder_few", kind="reorder", groups=1, width=4, layers=1, kv=5, dim=128, length=300, room=512, form="four"),
        # eight requests of eight beams, six layers of bf16 caches
        dict(name="reorder_many", kind="reorder", groups=8, width=8, layers=6, kv=5, dim=128, length=1040, room=1536, form="bfloat16"),
    ]


def _between(rng, low, high):
    """A whole number, spread over the logarithm."""
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "select", "reorder"])
    dim = rng.choice([64, 96, 128, 128, 256])
    if kind == "store":
        batch, kv = _between(rng, 1, 16), rng.randint(1, 8)
        seq = _between(rng, 1, max(1, 10000000 // (batch * kv * dim)))
        past = _between(rng, 1, 4000) - 1
        return dict(kind=kind, batch=batch, seq=seq, kv=kv, dim=dim, past=past, room=past + seq + rng.randint(0, 99),
                    dtype=rng.choice(list(TYPES)), stacked=rng.random() < 0.5)
    if kind == "attend":
        kv, each, batch = rng.randint(1, 8), rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), _between(rng, 1, 64)
        seq = rng.choice([1, 1, 1, 2, rng.randint(3, 40), _between(rng, 50, 1000)])
        batch = min(batch, max(1, 40000000000 // (kv * each * seq * dim * 2 * seq)))
        cells = min(270000000 // (batch * kv * dim), 40000000000 // (batch * kv * each * seq * dim))
        high = _between(rng, 16, max(17, min(131000, cells)))
        return dict(kind=kind, batch=batch, seq=seq, heads=kv * each, kv=kv, dim=dim, low=rng.choice([high, high // 3, 0]), high=high,
                    window=rng.choice([0, 0, 0, _between(rng, 1, 4096)]), sinks=rng.random() < 0.3, dtype=rng.choice(list(TYPES)))
    if kind == "select":
        groups, width = _between(rng, 1, 24), rng.randint(1, 12)
        vocab = _between(rng, 300, min(200000, 16000000 // (groups * width)))
        return dict(kind=kind, groups=groups, width=width, vocab=vocab, count=rng.randint(1, 2 * width), ended=rng.randint(0, width // 3),
                    dtype=rng.choice(list(TYPES)))
    groups, width, layers, length = _between(rng, 1, 12), rng.randint(2, 10), rng.randint(1, 6), _between(rng, 1, 2000)
    length = min(length, 120000000 // (groups * width * layers * dim))
    kv = rng.randint(1, max(1, min(8, 120000000 // (groups * width * layers * length * dim))))
    return dict(kind=kind, groups=groups, width=width, layers=layers, kv=kv, dim=dim, length=length, room=length + rng.randint(0, 200),
                form=rng.choice(["four", "bfloat16", "float32"]))


# ------------------------------------------------------------------ inputs
def _room(positions):
    return -(-positions // 16) * 16


def _past(case):
    """Cached lengths of the sequences: spread evenly between the case's bounds, in an order that mixes them."""
    n, low, high = case["batch"], case["low"], case["high"]
    return [low + (high - low) * ((7 * b + 3) % n) // max(1, n - 1) for b in range(n)]


def _rows(g, shape, dtype):
    """Keys or values as a model makes them: normal, with an offset and a size per head and column."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    size = torch.rand(shape[2:], generator=g, device="cuda") * 1.5 + 0.25
    offset = torch.randn(shape[2:], generator=g, device="cuda")
    return x.mul_(size).add_(offset).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return globals()["_prepare_" + case["kind"]](case, g)


def _new_cache(batch, kv, room, dim):
    """What a program keeps for a layer: the framework's cache, or the plain form's tensors of codes (two a byte), steps and
    smallest values."""
    if own:
        from rotor_b200.cache4 import Cache4
        return Cache4(batch, kv, room, dim)
    one = lambda n, t: torch.zeros((batch, kv, _room(room), n), dtype=t, device="cuda")
    return [[one(dim // 2, torch.uint8), one(dim // GROUP, torch.float16), one(dim // GROUP, torch.float16)] for _ in range(2)]


def _store_inputs(case, g):
    b, s, h, d, dtype = case["batch"], case["seq"], case["kv"], case["dim"], TYPES[case["dtype"]]
    k, v = _rows(g, (b, s, h, d), dtype), _rows(g, (b, s, h, d), dtype)
    if case["stacked"]:       # [queries | keys | values] of a token, four query heads per key/value head
        row = torch.zeros((b, s, 6 * h, d), dtype=dtype, device="cuda")
        row[:, :, 4 * h:5 * h], row[:, :, 5 * h:] = k, v
        k, v = row[:, :, 4 * h:5 * h], row[:, :, 5 * h:]
    return dict(kind="store", k=k, v=v, past=case["past"], seq=s, dtype=dtype)


def _prepare_store(case, g):
    return dict(_store_inputs(case, g), cache=_new_cache(case["batch"], case["kv"], case["room"], case["dim"]))


def _attend_inputs(case, g):
    b, s, h, d, past = case["batch"], case["seq"], case["kv"], case["dim"], _past(case)
    k, v = (_rows(g, (b, max(past) + s, h, d), torch.bfloat16) for _ in range(2))
    q = torch.randn((b, s, case["heads"], d), generator=g, device="cuda").to(TYPES[case["dtype"]])
    sinks = torch.randn(case["heads"], generator=g, device="cuda") if case["sinks"] else None
    even = min(past) == max(past)
    return k, v, dict(kind="attend", q=q, past=past[0] if even else torch.tensor(past, dtype=torch.int32, device="cuda"),
                      longest=max(past), window=case["window"], sinks=sinks, scale=1 / math.sqrt(d))


def _prepare_attend(case, g):
    k, v, state = _attend_inputs(case, g)
    state["cache"] = cache = _new_cache(k.shape[0], k.shape[2], k.shape[1], k.shape[3])
    if own:
        cache.append(k, v, 0)
    else:
        _append(cache, k, v, 0)
    return state


def _prepare_select(case, g):
    n, w, vocab = case["groups"], case["width"], case["vocab"]
    logits = torch.randn((n, w, vocab), generator=g, device="cuda").mul_(2.5).to(TYPES[case["dtype"]])
    scores = torch.rand((n, w), generator=g, device="cuda").mul_(-4).sub_(10)
    ended = torch.zeros((n, w), dtype=torch.bool, device="cuda")
    ended[:, w - case["ended"]:] = True
    return dict(kind="select", logits=logits, scores=scores, ended=ended if case["ended"] else None, count=case["count"], pad=vocab // 2)


def _prepare_reorder(case, g):
    n, w, d, room = case["groups"], case["width"], case["dim"], case["room"]
    if case["form"] == "four":       # codes, steps and smallest values of keys and of values
        forms = [(d // 2, torch.uint8), (d // GROUP, torch.float16), (d // GROUP, torch.float16)] * 2
    else:
        forms = [(d, TYPES[case["form"]])] * 2
    states = []
    for _ in range(case["layers"]):
        for columns, dtype in forms:
            shape = (n * w, case["kv"], _room(room), columns)
            if dtype is torch.uint8:
                states.append(torch.randint(0, 256, shape, generator=g, device="cuda", dtype=dtype))
            else:
                states.append(torch.randn(shape, generator=g, device="cuda", dtype=dtype))
    # half of the beams go on where they are and the others follow one of them each (so a pass can be repeated)
    order = torch.rand((n, w), generator=g, device="cuda").argsort(1)
    beams = torch.arange(w, device="cuda").repeat(n, 1)
    kept = w - w // 2
    beams.scatter_(1, order[:, kept:], order[:, :w // 2])
    return dict(kind="reorder", states=states, beams=beams, length=case["length"])


# ------------------------------------------------------------------ the operators
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["kind"]](state)


def _own_store(t):
    t["cache"].append(t["k"], t["v"], t["past"])
    return t["cache"].read(t["past"], t["past"] + t["seq"], dtype=t["dtype"])


def _own_attend(t):
    return t["cache"].attend(t["q"], t["past"], scale=t["scale"], window=t["window"], sinks=t["sinks"], longest=t["longest"])


def _own_select(t):
    from rotor_b200 import ops
    return ops.beam_select(t["logits"], t["scores"], t["count"], ended=t["ended"], pad=t["pad"])


def _own_reorder(t):
    from rotor_b200 import ops
    ops.reorder_states([(x, 2) for x in t["states"]], t["beams"], length=t["length"])
    return t["states"]


def _quantise(x):
    """Codes (float64), steps and smallest values (float16) of rows [..., dim].  A code is decided in 64 bits: it lies next to a
    border for many inputs of few bits."""
    x = x.float().clamp(-65504, 65504).unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step, least = ((high.double() - low.double()) / 15).float().half(), low.half()
    codes = ((x.double() - least.double()) / step.double()).round().clamp(0, 15)
    return torch.where(step > 0, codes, 0.0).flatten(-2), step.squeeze(-1), least.squeeze(-1)


def _append(cache, k, v, past):
    for x, (codes, steps, least) in zip((k, v), cache):
        at = slice(past, past + x.shape[1])
        q, s, m = _quantise(x.transpose(1, 2))
        q = q.to(torch.uint8)
        codes[:, :, at], steps[:, :, at], least[:, :, at] = q[..., 0::2] | q[..., 1::2] << 4, s, m


def _values(part, at):
    """The values that the positions ``at`` of a part of the cache stand for, in float32."""
    codes, steps, least = (x[:, :, at] for x in part)
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    return (q * steps.float()[..., None] + least.float()[..., None]).flatten(-2)


def _plain_store(t):
    _append(t["cache"], t["k"], t["v"], t["past"])
    at = slice(t["past"], t["past"] + t["seq"])
    return tuple(_values(part, at).to(t["dtype"]) for part in t["cache"])


def _plain_attend(t):
    q = t["q"]
    b, s, heads, d = q.shape
    total = t["longest"] + s
    k, v = (_values(part, slice(0, total)) for part in t["cache"])
    h = k.shape[1]
    rows = q.float().unflatten(2, (h, heads // h)).permute(0, 2, 3, 1, 4)                        # b h g s d
    x = (rows.reshape(b, h, -1, d) @ k.transpose(2, 3)).unflatten(2, (heads // h, s)) * t["scale"]  # b h g s t
    past = torch.as_tensor(t["past"], device=q.device).reshape(-1, 1, 1)
    i, j = past + torch.arange(s, device=q.device)[None, :, None], torch.arange(total, device=q.device)
    seen = (j <= i) & ((i - j < t["window"]) if t["window"] else torch.ones_like(j, dtype=torch.bool))
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    sink = None if t["sinks"] is None else t["sinks"].reshape(1, h, -1, 1, 1)
    if sink is not None:
        top = torch.maximum(top, sink)
    x = (x - top).exp()
    mass = x.sum(-1, keepdim=True)
    if sink is not None:
        mass = mass + (sink - top).exp()
    y = (x.reshape(b, h, -1, total) @ v).unflatten(2, (heads // h, s)) / mass
    return y.permute(0, 3, 1, 2, 4).reshape(b, s, heads, d).to(q.dtype)


def _plain_select(t):
    """In 64 bits: candidates of different beams lie close to one another."""
    x, scores = t["logits"].double(), t["scores"].double()[..., None]
    top = x.amax(-1, keepdim=True)
    x = scores + (x - (top + (x - top).exp().sum(-1, keepdim=True).log()))
    if t["ended"] is not None:
        goes_on = ~t["ended"][..., None]
        only = torch.arange(x.shape[-1], device=x.device) == t["pad"]
        x = torch.where(goes_on, x, torch.where(only, scores, -math.inf))
    best, at = x.flatten(1).sort(dim=1, descending=True, stable=True)
    best, at = best[:, :t["count"]], at[:, :t["count"]]
    return best.float(), at // x.shape[-1], at % x.shape[-1]


def _plain_reorder(t):
    n, w = t["beams"].shape
    rows = (t["beams"] + w * torch.arange(n, device="cuda")[:, None]).flatten()
    for x in t["states"]:
        x[:, :, :t["length"]] = x[:, :, :t["length"]][rows]
    return t["states"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    return globals()["_work_" + case["kind"]](case)


def _size(name):
    return {"float32": 4}.get(name, 2)


def _row_bytes(dim):
    """One position of one head, key or value: codes, steps, smallest values."""
    return dim // 2 + 4 * (dim // GROUP)


def _work_store(c):
    rows = 2 * c["batch"] * c["seq"] * c["kv"]
    return {"bytes": rows * (2 * c["dim"] * _size(c["dtype"]) + 2 * _row_bytes(c["dim"])), "flops": rows * c["dim"] * 8}


def _work_attend(c):
    rows = pairs = 0
    for past in _past(c):
        first = max(0, past - c["window"] + 1) if c["window"] else 0
        rows += past + c["seq"] - first
        pairs += sum(min(p + 1, c["window"] or p + 1) for p in range(past, past + c["seq"]))
    q = c["batch"] * c["seq"] * c["heads"] * c["dim"] * _size(c["dtype"])
    return {"bytes": 2 * c["kv"] * rows * _row_bytes(c["dim"]) + 2 * q, "flops": 4 * c["heads"] * c["dim"] * pairs}


def _work_select(c):
    n = c["groups"] * (c["width"] - c["ended"]) * c["vocab"]
    return {"bytes": n * _size(c["dtype"]) + c["groups"] * (4 * c["width"] + 20 * c["count"]), "flops": 4 * n}


def _work_reorder(c):
    row = 2 * _row_bytes(c["dim"]) if c["form"] == "four" else 2 * c["dim"] * _size(c["form"])
    moved = c["groups"] * (c["width"] // 2)
    return {"bytes": 2 * moved * c["layers"] * c["kv"] * c["length"] * row + 8 * c["groups"] * c["width"], "flops": 0}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    """From the inputs alone.  States that are moved are compared as they are."""
    kind, g = case["kind"], torch.Generator(device="cuda").manual_seed(seed)
    if kind == "store":
        t = _store_inputs(case, g)
        return tuple(_exact_values(x).transpose(1, 2) for x in (t["k"], t["v"]))
    if kind == "attend":
        k, v, t = _attend_inputs(case, g)
        return _exact_attend(t, _exact_values(k), _exact_values(v))
    if kind == "select":
        return _exact_select(_prepare_select(case, g))
    t = _prepare_reorder(case, g)
    width, length, out = case["width"], case["length"], []
    for x in t["states"]:
        y = x.clone()
        for row, source in enumerate(t["beams"].flatten().tolist()):
            y[row, :, :length] = x[row // width * width + source, :, :length]
        out.append(y.double() if y.dtype.is_floating_point else y)
    return out


def _exact_values(x):
    """What the cache holds of rows [..., dim]: every column's nearest level, the even one of two as near."""
    x = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP).clip(-65504.0, 65504.0)
    low, high = torch.aminmax(x, dim=-1, keepdim=True)
    m = low.to(torch.float32).to(torch.float16).double()
    s = ((high - low) / 15.0).to(torch.float32).to(torch.float16).double()
    u = (x - m) / s.masked_fill(s == 0, 1.0)
    below = torch.floor(u)
    rest = u - below
    up = (rest > 0.5) | ((rest == 0.5) & (below % 2 == 1))
    code = (below + up).clip(0, 15) * (s != 0)
    return (m + s * code).reshape(*x.shape[:-2], -1)


def _exact_attend(t, k, v):
    q = t["q"].double() * t["scale"]
    b, s, heads, d = q.shape
    h = k.shape[2]
    out = torch.empty_like(q)
    past = t["past"].tolist() if torch.is_tensor(t["past"]) else [t["past"]] * b
    for n in range(b):
        for head in range(heads):
            keys, values = k[n, :, head // (heads // h)], v[n, :, head // (heads // h)]
            x = q[n, :, head] @ keys.T
            at = torch.arange(past[n], past[n] + s, device=x.device)[:, None] - torch.arange(keys.shape[0], device=x.device)
            hidden = at < 0 if not t["window"] else (at < 0) | (at >= t["window"])
            x[hidden] = -math.inf
            if t["sinks"] is not None:
                sink = t["sinks"][head].double().expand(s, 1)
                out[n, :, head] = torch.softmax(torch.cat([x, sink], 1), 1)[:, :-1] @ values
            else:
                out[n, :, head] = torch.softmax(x, 1) @ values
    return out


def _exact_select(t):
    n, w, vocab = t["logits"].shape
    scores, beams, tokens = [], [], []
    for i in range(n):
        x = torch.log_softmax(t["logits"][i].double(), -1) + t["scores"][i].double()[:, None]
        if t["ended"] is not None:
            x[t["ended"][i]] = -math.inf
            x[t["ended"][i], t["pad"]] = t["scores"][i][t["ended"][i]].double()
        order = torch.argsort(-x.reshape(-1), stable=True)[:t["count"]]
        scores.append(x.reshape(-1)[order])
        beams.append(torch.div(order, vocab, rounding_mode="floor"))
        tokens.append(order.remainder(vocab))
    return torch.stack(scores), torch.stack(beams), torch.stack(tokens)
