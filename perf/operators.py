"""The operators of a batched decode step that are measured: products with 4-bit weights and group scales, the
selection of a beam search over the beams' logits, and the reordering of the beams' states.

Every operator has a plain form (elementary torch operations) and the framework's own calls, chosen by ``own``."""
import math

import numpy as np
import torch

own = False

_T = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int64": torch.int64}


# ------------------------------------------------------------------------------------------------------ cases
def listed():
    lin = dict(op="linear", x="bf16", out="bf16", scales="fp32", bias=False)
    beam = dict(op="select", finished=False, first=False, tail=0)
    return [
        # one token through a square projection of a small model: latency
        dict(lin, name="nf4 4096x4096 1 row", rows=1, n=4096, k=4096, group=64, kind="code"),
        # one token through an attention projection of the 126-layer stack
        dict(lin, name="nf4 16384x16384 1 row", rows=1, n=16384, k=16384, group=64, kind="code"),
        # odd sizes, a last group that is not full, zero points, a bias
        dict(lin, name="int4 1001x2086 3 rows", rows=3, n=1001, k=2086, group=128, kind="zeros", x="fp16", out="fp16",
             scales="fp16", bias=True),
        # a batch of eight through an MLP projection, zero points for each group
        dict(lin, name="int4 14336x4096 8 rows", rows=8, n=14336, k=4096, group=128, kind="zeros", scales="bf16"),
        # four beams through an NF4 vocabulary head, logits in 32 bits
        dict(lin, name="nf4 128256x4096 4 rows", rows=4, n=128256, k=4096, group=64, kind="code", out="fp32"),
        # the widest projection of the 126-layer stack with 32 rows (four prompts of eight beams)
        dict(lin, name="int4 53248x16384 32 rows", rows=32, n=53248, k=16384, group=128, kind="sym", scales="fp16"),
        # the first step of one prompt: only beam 0 is alive
        dict(beam, name="select 1x4 first step", batch=1, beams=4, vocab=128256, cand=8, x="fp32", first=True),
        # an odd vocabulary in a padded buffer, some beams finished
        dict(beam, name="select 24x5 vocab 50257", batch=24, beams=5, vocab=50257, cand=5, x="fp16", finished=True, tail=47),
        # a serving batch with logits in 16 bits
        dict(beam, name="select 16x8 bf16", batch=16, beams=8, vocab=128256, cand=16, x="bf16"),
        # the largest batch, logits in 32 bits
        dict(beam, name="select 32x16 fp32", batch=32, beams=16, vocab=128256, cand=32, x="fp32", finished=True),
        # one prompt's residual and token history
        dict(op="reorder", name="reorder 1x4 small", batch=1, beams=4, tensors=2, heads=1, max_len=511, length=511, dim=8,
             x="fp32"),
        # the keys and values of eight layers at 1500 of 2048 positions
        dict(op="reorder", name="reorder 4x8 caches", batch=4, beams=8, tensors=16, heads=8, max_len=2048, length=1500,
             dim=128, x="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear", "select", "select", "reorder"))
    if op == "linear":
        n, k = _log(rng, 16, 65536), 2 * _log(rng, 32, 8192)
        if rng.random() < 0.5:
            n, k = max(16, n // 16 * 16), max(64, k // 64 * 64)
        n = min(n, 53248 * 16384 // k)
        x = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        return dict(op=op, rows=_log(rng, 1, 32), n=n, k=k, group=rng.choice((32, 64, 64, 128, 128, 256)),
                    kind=rng.choice(("code", "code", "sym", "zeros")), x=x, out=rng.choice((x, x, "fp32")),
                    scales=rng.choice(("fp32", "fp16", "bf16")), bias=rng.random() < 0.3)
    if op == "select":
        batch, beams = _log(rng, 1, 32), rng.randint(1, 16)
        return dict(op=op, batch=batch, beams=beams, vocab=_log(rng, 500, 128256), cand=rng.randint(1, 2 * beams),
                    x=rng.choice(("fp32", "fp16", "bf16")), finished=rng.random() < 0.4, first=rng.random() < 0.2,
                    tail=rng.choice((0, 0, 3, 64)))
    c = dict(op=op, batch=_log(rng, 1, 6), beams=rng.randint(2, 8), tensors=rng.randint(1, 12), heads=rng.randint(1, 8),
             dim=rng.choice((3, 64, 80, 128)), x=rng.choice(("bf16", "fp16", "fp32", "int64")))
    each = c["batch"] * c["beams"] * c["tensors"] * c["heads"] * c["dim"] * (8 if c["x"] == "int64" else 4)
    c["max_len"] = _log(rng, 16, min(2048, (1 << 30) // each))
    return dict(c, length=rng.randint(max(1, c["max_len"] // 4), c["max_len"]))


# ----------------------------------------------------------------------------------------------------- inputs
def _normal_code(dev):
    """16 values in [-1, 1] at the quantiles of a normal distribution, zero among them (the 4-bit codebook of QLoRA)."""
    p = torch.linspace(0.9677083, 0.5, 9, dtype=torch.float64)[:-1]
    q = torch.linspace(0.9677083, 0.5, 8, dtype=torch.float64)[:-1]
    v = torch.cat([torch.special.ndtri(p), torch.zeros(1, dtype=torch.float64), -torch.special.ndtri(q)]).sort().values
    return (v / v.max()).float().to(dev)


def _prepare_linear(c, gen, dev):
    n, k, g = c["n"], c["k"], -(-c["k"] // c["group"])
    s = {"packed": torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=dev, generator=gen)}
    spread = torch.rand((n, g), device=dev, generator=gen)
    code = c["kind"] == "code"
    s["scales"] = ((0.03 + 0.04 * spread) * (1.0 if code else 1 / 7.5)).to(_T[c["scales"]])
    s["code"] = _normal_code(dev) if code else None
    s["zeros"] = torch.randint(4, 12, (n, g), dtype=torch.uint8, device=dev, generator=gen) if c["kind"] == "zeros" else None
    s["bias"] = (torch.randn(n, device=dev, generator=gen) * 0.3).to(_T[c["x"]]) if c["bias"] else None
    x = torch.randn((c["rows"], k), device=dev, generator=gen)
    x[:, :: max(2, k // 7)] *= 20.0  # a few channels of a hidden state are far larger than the others
    s["x"] = x.to(_T[c["x"]])
    if own:  # the layer that a user's program builds once, when it loads its weights
        from next_step_ai_b200.linear4bit import Linear4bit
        s["layer"] = Linear4bit(s["packed"], s["scales"], out_features=n, in_features=k, group_size=c["group"],
                                code=s["code"], zeros=s["zeros"], bias=s["bias"])
    return s


def _prepare_select(c, gen, dev):
    b, w, v = c["batch"], c["beams"], c["vocab"]
    x = torch.randn((b, w, v + c["tail"]), device=dev, generator=gen) * 2.5
    x -= 1.5 * torch.log1p(torch.arange(v + c["tail"], device=dev) / 64.0)[torch.randperm(v + c["tail"], device=dev, generator=gen)]
    x[..., torch.randint(0, v, (max(1, v // 100),), device=dev, generator=gen)] = -math.inf  # words that may not come
    s = {"buffer": x.to(_T[c["x"]])}
    s["logits"] = s["buffer"][..., :v]  # the vocabulary's padding is no part of the logits
    s["scores"] = -20.0 * torch.rand((b, w), device=dev, generator=gen)
    if c["first"]:
        s["scores"][:, 1:] = -math.inf
    s["finished"] = torch.rand((b, w), device=dev, generator=gen) < 0.25 if c["finished"] else None
    return s


def _parents(c, seed):
    """Whose state each beam goes on with: of the same shape for every seed, at other places."""
    r, w = np.random.default_rng(seed), c["beams"]
    base = np.arange(w)
    base[w // 2:] = base[w // 2:] - w // 2 if w % 2 == 0 else base[w // 2:] // 2  # half go on with another's state
    rows = []
    for _ in range(c["batch"]):
        p = r.permutation(w)
        row = np.empty(w, np.int64)
        row[p] = p[base]
        rows.append(row)
    return np.stack(rows)


def _reorder_shapes(c):
    """(shape, the dimension of the positions)"""
    rows = c["batch"] * c["beams"]
    if c["heads"] == 1 and c["dim"] <= 8:
        return [((rows, c["max_len"] * c["dim"]), None), ((rows, c["max_len"]), 1)][: c["tensors"]]
    return [((rows, c["heads"], c["max_len"], c["dim"]), 2)] * c["tensors"]


def _prepare_reorder(c, gen, dev, seed):
    kind = _T[c["x"]]
    shapes = _reorder_shapes(c)
    s = {"states": [torch.randint(0, 1 << 15, sh, device=dev, generator=gen) if kind == torch.int64
                    else torch.randn(sh, device=dev, generator=gen, dtype=kind) for sh, _ in shapes]}
    s["dims"], s["length"], s["parents"] = [d for _, d in shapes], c["length"], torch.from_numpy(_parents(c, seed)).to(dev)
    if own:  # the handle that a user's program builds once, for its caches
        from next_step_ai_b200.beam import BeamStates
        s["handle"] = BeamStates(s["states"], batch=c["batch"], beams=c["beams"], length_dims=s["dims"])
    return s


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    c = dict(case)
    if c["op"] == "linear":
        s = _prepare_linear(c, gen, dev)
    elif c["op"] == "select":
        s = _prepare_select(c, gen, dev)
    else:
        s = _prepare_reorder(c, gen, dev, seed)
    return dict(s, case=c)


# ------------------------------------------------------------------------------------------------ plain forms
def _linear(s):
    c = s["case"]
    q = torch.stack([s["packed"] >> 4, s["packed"] & 15], dim=-1).reshape(c["n"], c["k"])
    g = s["scales"].shape[1]
    w = s["code"][q.int()] if s["code"] is not None else q.float()
    w = torch.nn.functional.pad(w, (0, g * c["group"] - c["k"])).reshape(c["n"], g, c["group"])
    if s["code"] is None:
        w = w - (s["zeros"].float()[..., None] if s["zeros"] is not None else 8.0)
    w = (w * s["scales"].float()[..., None]).reshape(c["n"], -1)[:, : c["k"]]
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(_T[c["out"]])


def _select(s):
    """Scores in 64 bits, since beams are compared by sums that may be near to each other."""
    c = s["case"]
    b, w, v, k = c["batch"], c["beams"], c["vocab"], min(c["cand"], c["vocab"])
    x = s["logits"].float()
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)  # as the values are ordered
    key = order * (1 << 31) + (v - 1 - torch.arange(v, device=x.device))  # of equal ones the first comes first
    at = v - 1 - (torch.topk(key, k, dim=-1).values & 0x7FFFFFFF)
    d = x.double()
    top = d.amax(dim=-1, keepdim=True)
    lse = top + torch.log(torch.exp(d - top).sum(dim=-1, keepdim=True))
    got = s["scores"].double()[..., None] + (torch.gather(d, -1, at) - lse)
    if s["finished"] is not None:  # a finished beam goes on as it is, with token 0
        f = s["finished"][..., None]
        first = torch.arange(k, device=x.device) == 0
        got = torch.where(f, torch.where(first, s["scores"].double()[..., None], -math.inf), got)
        at = torch.where(f, torch.where(first, 0, torch.arange(k, device=x.device)), at)
    flat = (at + v * torch.arange(w, device=x.device)[:, None]).reshape(b, w * k)
    flat, by = torch.sort(flat, dim=-1)
    got, by = torch.sort(torch.gather(got.reshape(b, w * k), -1, by), dim=-1, descending=True, stable=True)
    flat, got = torch.gather(flat, -1, by)[:, : c["cand"]], got[:, : c["cand"]]
    more = c["cand"] - flat.shape[1]
    flat, got = torch.nn.functional.pad(flat, (0, more)), torch.nn.functional.pad(got, (0, more), value=-math.inf)
    none = got == -math.inf
    return got.float(), torch.where(none, -1, flat % v), torch.where(none, 0, flat // v)


def _reorder(s):
    c = s["case"]
    rows = (s["parents"] + c["beams"] * torch.arange(c["batch"], device=s["parents"].device)[:, None]).reshape(-1)
    live = [t if d is None else t.narrow(d, 0, c["length"]) for t, d in zip(s["states"], s["dims"])]
    [t.copy_(t[rows]) for t in live]
    return s["states"]


def run(s):
    c = s["case"]
    if not own:
        return {"linear": _linear, "select": _select, "reorder": _reorder}[c["op"]](s)
    if c["op"] == "linear":
        return s["layer"](s["x"], out_dtype=_T[c["out"]])
    if c["op"] == "select":
        from next_step_ai_b200.beam import beam_select
        return beam_select(s["logits"], s["scores"], num_candidates=c["cand"], finished=s["finished"], pad_token=0)
    s["handle"].reorder_(s["parents"], length=s["length"])
    return s["states"]


# ------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    size = {"fp32": 4, "fp16": 2, "bf16": 2, "int64": 8}
    if c["op"] == "linear":
        n, k, g, t = c["n"], c["k"], -(-c["k"] // c["group"]), c["rows"]
        weights = n * k // 2 + n * g * (size[c["scales"]] + (1 if c["kind"] == "zeros" else 0)) + (64 if c["kind"] == "code" else 0)
        return {"bytes": weights + t * k * size[c["x"]] + t * n * size[c["out"]] + (n * size[c["x"]] if c["bias"] else 0),
                "flops": 2.0 * t * n * k}
    if c["op"] == "select":
        rows = c["batch"] * c["beams"]
        alive = rows * (0.75 if c["finished"] else 1.0)
        if c["first"]:  # the rows of beams that are out need not be read
            alive /= c["beams"]
        return {"bytes": alive * c["vocab"] * size[c["x"]] + rows * 4 + c["batch"] * c["cand"] * 20,
                "flops": alive * c["vocab"] * 4.0}
    p = _parents(c, 1)  # as many moves for every seed
    moved = int((p != np.arange(c["beams"])).sum())
    read = sum(len(set(r[r != np.arange(c["beams"])])) for r in p)
    each = 0
    for sh, d in _reorder_shapes(c):
        each += math.prod(sh[1:]) * size[c["x"]] if d is None else math.prod(sh[1:]) // sh[d] * c["length"] * size[c["x"]]
    return {"bytes": (moved + read) * each + p.size * 8, "flops": 0.0}


# ---------------------------------------------------------------------------------------------- in 64 bits
def _exact_linear(c, seed):
    s = prepare(c, seed)
    x = s["x"].double()
    out = []
    for r in range(0, c["n"], 4096):  # the even and the odd columns apart: the two halves of each byte
        p = s["packed"][r: r + 4096]
        sc = s["scales"][r: r + 4096].double()
        z = s["zeros"][r: r + 4096].double() if s["zeros"] is not None else torch.full_like(sc, 8.0)
        group = torch.arange(p.shape[1], device=p.device) * 2 // c["group"]  # groups are even: both columns are in one
        table = s["code"].double() if s["code"] is not None else torch.arange(16, device=p.device).double()
        y = 0.0
        for half, nib in ((0, p // 16), (1, p % 16)):
            w = table[nib.long()]
            if s["code"] is None:
                w -= z[:, group]
            y = y + x[:, half::2] @ (w.mul_(sc[:, group])).t()
        out.append(y)
    y = torch.cat(out, dim=1)
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_select(c, seed):
    s = prepare(c, seed)
    v, fin = c["vocab"], s["finished"]
    scores, tokens, parents = [], [], []
    for b in range(c["batch"]):
        d = torch.log_softmax(s["logits"][b].double(), dim=-1) + s["scores"][b].double()[:, None]
        if fin is not None:
            d[fin[b]] = -math.inf
            d[fin[b], 0] = s["scores"][b].double()[fin[b]]
        d = d.reshape(-1)
        val, at = torch.sort(d, descending=True, stable=True)
        val, at = val[: c["cand"]], at[: c["cand"]]
        gone = val == -math.inf
        scores.append(val)
        tokens.append(at.remainder(v).masked_fill(gone, -1))
        parents.append(at.div(v, rounding_mode="floor").masked_fill(gone, 0))
    return torch.stack(scores), torch.stack(tokens), torch.stack(parents)


def _exact_reorder(c, seed):
    s = prepare(c, seed)
    src = s["parents"].cpu().numpy()
    for t, d in zip(s["states"], s["dims"]):
        old = t.clone()
        for b in range(c["batch"]):
            for j in range(c["beams"]):
                to, frm = t[b * c["beams"] + j], old[b * c["beams"] + int(src[b, j])]
                if d is None:
                    to.copy_(frm)
                else:
                    to.narrow(d - 1, 0, c["length"]).copy_(frm.narrow(d - 1, 0, c["length"]))
    return [t.double() if t.is_floating_point() else t for t in s["states"]]


def exact(case, seed):
    c = dict(case)
    return {"linear": _exact_linear, "select": _exact_select, "reorder": _exact_reorder}[c["op"]](c, seed)
