"""The per-head rotation and the windowed attention of a single-sequence track, as cases to time.

A program that runs such a track keeps two operators for each layer: HeadRotary, which norms the queries and
keys of each head, turns them by their positions and writes keys and values into the layer's cache, and
WindowAttention, which attends over a window of the last keys and the first few ("sinks"). The kinds:

  rotary           q and k of a prompt or of single tokens, with the norm of each head; k and v into a cache
  rotary_backward  the gradients of q, k and of the norms' weights
  attention        a prompt, a piece of one, or single tokens against a cache; outputs and log-sum-exps
  attention_backward  the gradients of q, k and v

"f16" is what a deployment runs, "f32" the framework's default. Sequences of a batch have lengths of their own;
tensors are [batch][tokens][heads][channels]. Widths are those of this repository's attention (8 heads of 32)
and generic ones (32 heads over 8 of keys, 128 channels each). A window of -1 has no end on that side.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

EPS = 1e-5
DTYPE = {"f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------

def listed() -> list:
    return [
        # The smallest call: one token for each of eight sequences, every layer of every step. Latency counts.
        {"name": "rotary_step_f16", "kind": "rotary", "dtype": "f16", "batch": 8, "tokens": 1, "heads": 32,
         "key_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "norm": "rms", "scaling": "none",
         "capacity": 512, "ragged": True},
        # Two long prompts, into an empty cache.
        {"name": "rotary_prompt_f16", "kind": "rotary", "dtype": "f16", "batch": 2, "tokens": 4096, "heads": 32,
         "key_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "norm": "rms", "scaling": "yarn",
         "capacity": 4096, "ragged": False},
        # A padded batch at the default precision: odd length, narrow heads, half of the channels turned, no cache.
        {"name": "rotary_odd_f32", "kind": "rotary", "dtype": "f32", "batch": 3, "tokens": 1021, "heads": 8,
         "key_heads": 8, "dim": 32, "rotary": 16, "layout": "interleaved", "norm": "layer", "scaling": "linear",
         "capacity": 0, "ragged": True},
        # The training step's way back through it.
        {"name": "rotary_backward_f16", "kind": "rotary_backward", "dtype": "f16", "batch": 1, "tokens": 4096,
         "heads": 32, "key_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "norm": "rms", "scaling": "none",
         "ragged": False},
        # A step of sixteen sequences in a layer with a window: a few MB of the cache are visible.
        {"name": "step_window_f16", "kind": "attention", "dtype": "f16", "batch": 16, "queries": 1, "keys": 4096,
         "heads": 32, "key_heads": 8, "dim": 128, "left": 1023, "right": 0, "sinks": 4, "ragged": True},
        # A step of four sequences in a layer without one, over a long cache: bandwidth counts.
        {"name": "step_long_f16", "kind": "attention", "dtype": "f16", "batch": 4, "queries": 1, "keys": 32768,
         "heads": 32, "key_heads": 8, "dim": 128, "left": -1, "right": 0, "sinks": 0, "ragged": True},
        # The next piece of a long prompt against what is in the cache.
        {"name": "piece_f16", "kind": "attention", "dtype": "f16", "batch": 1, "queries": 256, "keys": 8192,
         "heads": 32, "key_heads": 8, "dim": 128, "left": 4095, "right": 0, "sinks": 4, "ragged": False},
        # A whole prompt without a window.
        {"name": "prompt_f16", "kind": "attention", "dtype": "f16", "batch": 1, "queries": 4096, "keys": 4096,
         "heads": 32, "key_heads": 8, "dim": 128, "left": -1, "right": 0, "sinks": 0, "ragged": False},
        # A long prompt with a window: most of the square is never visited.
        {"name": "prompt_window_f16", "kind": "attention", "dtype": "f16", "batch": 1, "queries": 16384,
         "keys": 16384, "heads": 8, "key_heads": 2, "dim": 128, "left": 1023, "right": 0, "sinks": 4,
         "ragged": False},
        # Sequence-local attention, both ways, over a padded batch of chains at the default precision.
        {"name": "local_f32", "kind": "attention", "dtype": "f32", "batch": 4, "queries": 1023, "keys": 1023,
         "heads": 8, "key_heads": 8, "dim": 32, "left": 128, "right": 128, "sinks": 0, "ragged": True},
        # Training with a window, f16.
        {"name": "backward_f16", "kind": "attention_backward", "dtype": "f16", "batch": 1, "queries": 4096,
         "keys": 4096, "heads": 16, "key_heads": 4, "dim": 128, "left": 1023, "right": 0, "sinks": 4,
         "ragged": False},
        # Training of the sequence-local attention at the default precision.
        {"name": "backward_local_f32", "kind": "attention_backward", "dtype": "f32", "batch": 2, "queries": 515,
         "keys": 515, "heads": 8, "key_heads": 8, "dim": 32, "left": 64, "right": 64, "sinks": 1, "ragged": True},
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "rotary", "rotary_backward", "attention", "attention", "attention", "attention",
                       "attention_backward", "attention_backward"])
    dtype = rng.choice(["f16", "f16", "f32"])
    heads, key_heads = rng.choice([(8, 8), (8, 2), (16, 4), (32, 8), (4, 1), (6, 3), (16, 1)])
    dim = rng.choice([32, 40, 64, 80, 128, 128])
    ragged = rng.random() < 0.6
    if kind in ("rotary", "rotary_backward"):
        single = kind == "rotary" and rng.random() < 0.4
        batch = _log(rng, 1, 64) if single else rng.choice([1, 2, 3])
        tokens = 1 if single else _log(rng, 5, 4000)
        case = {"kind": kind, "dtype": dtype, "batch": batch, "tokens": tokens, "heads": heads,
                "key_heads": key_heads, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]),
                "layout": rng.choice(["half", "interleaved"]), "norm": rng.choice(["none", "rms", "layer"]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "ragged": ragged}
        if kind == "rotary":
            case["capacity"] = tokens + _log(rng, 1, 400) if single or rng.random() < 0.5 else 0
        return case
    left, sinks = rng.choice([(-1, 0), (_log(rng, 30, 2000), rng.choice([0, 1, 4, 70])), (_log(rng, 30, 500), 4)])
    right = rng.choice([0, 0, _log(rng, 1, 300), -1])
    case = {"kind": kind, "dtype": dtype, "heads": heads, "key_heads": key_heads, "dim": dim, "left": left,
            "right": right, "sinks": sinks, "ragged": ragged}
    use = rng.choice(["step", "piece", "prompt", "prompt"]) if kind == "attention" else "prompt"
    if use == "step":
        case |= {"batch": _log(rng, 1, 32), "queries": 1, "keys": _log(rng, 20, 8000), "right": 0}
    elif use == "piece":
        queries = _log(rng, 2, 300)
        case |= {"batch": rng.choice([1, 2]), "queries": queries, "keys": queries + _log(rng, 20, 6000)}
    else:
        most = 1000 if dtype == "f32" else 2000 if kind == "attention" else 1200
        queries = _log(rng, 20, most)
        case |= {"batch": rng.choice([1, 2]), "queries": queries, "keys": queries}
    return case


def _lengths(case: dict) -> tuple:
    """The sequences' numbers of queries and of keys: the first whole, the others shorter where they are ragged."""
    if case["kind"].startswith("rotary"):
        queries, keys = case["tokens"], max(case["tokens"], case.get("capacity", 0))
    else:
        queries, keys = case["queries"], case["keys"]
    ql, kl = [], []
    for b in range(case["batch"]):
        cut = (b * 37 % 101) / 140 if case["ragged"] else 0.0
        q = queries if queries <= 1 else queries - int(queries * cut)
        ql.append(q)
        kl.append(max(q, keys - int(keys * cut)))
    return ql, kl


def _frequencies(case: dict) -> tuple:
    """(angle of one position for each turned pair, in 64 bits; the factor on what is turned)."""
    r = case["rotary"]
    base, factor, trained = 10000.0, 4.0, 2048
    at = torch.arange(0, r, 2, dtype=torch.float64) / r
    if case["scaling"] == "ntk":
        base *= factor ** (r / (r - 2))
    f = base ** -at
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] != "yarn":
        return f, 1.0
    # Pairs that turn often within the trained length stay, those that turn less than once are slowed.
    turns = trained * f / (2 * math.pi)
    keep = ((turns.log() - math.log(1.0)) / (math.log(32.0) - math.log(1.0))).clamp(0, 1)
    return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1.0


def _pairs(case: dict) -> int:
    """Visible (query, key) pairs of one head, over the batch."""
    total = 0
    for ql, kl in zip(*_lengths(case)):
        p = torch.arange(ql, dtype=torch.int64) + (kl - ql)
        high = (p + case["right"] + 1).clamp(0, kl) if case["right"] >= 0 else torch.full_like(p, kl)
        low = (p - case["left"]).clamp(min=0).minimum(high) if case["left"] >= 0 else torch.zeros_like(p)
        total += int((high - low + torch.minimum(low, torch.full_like(p, case["sinks"]))).sum())
    return total


def _keys_read(case: dict) -> int:
    total = 0
    for ql, kl in zip(*_lengths(case)):
        high = min(kl, kl + max(case["right"], 0))
        low = max(0, kl - ql - case["left"]) if case["left"] >= 0 else 0
        total += high - low + min(low, case["sinks"])
    return total


def work(case: dict) -> dict:
    es = 2 if case["dtype"] == "f16" else 4
    ql, kl = _lengths(case)
    h, hk, d = case["heads"], case["key_heads"], case["dim"]
    if case["kind"] == "rotary":
        values = sum(ql) * d * (h + hk + (hk if case["capacity"] else 0))
        return {"bytes": 2 * es * values, "flops": 10 * values}
    if case["kind"] == "rotary_backward":
        values = sum(ql) * d * (h + hk)
        return {"bytes": 3 * es * values, "flops": 20 * values}
    q, k = sum(ql) * h * d * es, _keys_read(case) * hk * d * es
    flops = 2 * d * h * _pairs(case)
    if case["kind"] == "attention":
        return {"bytes": 2 * q + 2 * k + 4 * sum(ql) * h, "flops": 2 * flops}
    return {"bytes": 4 * q + 4 * k + 4 * sum(ql) * h, "flops": 5 * flops}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPE[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dtype)

    b, h, hk, d = case["batch"], case["heads"], case["key_heads"], case["dim"]
    ql, kl = _lengths(case)
    s = {"case": case}
    lengths = torch.tensor(ql, dtype=torch.int32, device=dev)
    if case["kind"].startswith("rotary"):
        t = case["tokens"]
        # q, k and v lie side by side, as one projection writes them.
        qkv = normal(b, t, (h + 2 * hk) * d)
        s["q"] = qkv[..., :h * d].unflatten(-1, (h, d))
        s["k"] = qkv[..., h * d:(h + hk) * d].unflatten(-1, (hk, d))
        s["v"] = qkv[..., (h + hk) * d:].unflatten(-1, (hk, d))
        s["lengths"] = lengths if case["ragged"] and t > 1 else None
        # What the sequences hold before these tokens.
        past = [k - q for q, k in zip(ql, kl)]
        s["past"] = torch.tensor(past, dtype=torch.int32, device=dev) if any(past) else None
        s["frequencies"], s["turn"] = _frequencies(case)
        s["weights"] = None
        if case["norm"] != "none":
            s["weights"] = {"query_scale": 1 + normal(d, scale=0.1, dtype=torch.float32),
                            "key_scale": 1 + normal(d, scale=0.1, dtype=torch.float32)}
            if case["norm"] == "layer":
                s["weights"] |= {"query_offset": normal(d, scale=0.1, dtype=torch.float32),
                                 "key_offset": normal(d, scale=0.1, dtype=torch.float32)}
        if case["kind"] == "rotary" and case["capacity"]:
            s["k_cache"], s["v_cache"] = normal(b, case["capacity"], hk, d), normal(b, case["capacity"], hk, d)
        if case["kind"] == "rotary_backward":
            s["dq"], s["dk"] = normal(b, t, h, d), normal(b, t, hk, d)
    else:
        s["q"] = normal(b, case["queries"], h, d)
        s["k"], s["v"] = normal(b, case["keys"], hk, d), normal(b, case["keys"], hk, d)
        s["query_lengths"] = lengths if case["ragged"] and case["queries"] > 1 else None
        s["key_lengths"] = torch.tensor(kl, dtype=torch.int32, device=dev) if case["ragged"] else None
        if case["kind"] == "attention_backward":
            s["dout"] = normal(b, case["queries"], h, d)
            # What the forward pass left.
            s["out"], s["lse"] = _attend(s)
    if own:
        s["op"] = _operator(s)
    return s


def _operator(s: dict):
    path = os.path.join(os.getcwd(), "alphafold2-webgpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    case = s["case"]
    if case["kind"].startswith("rotary"):
        from afhip import rotary

        op = rotary.HeadRotary(case["heads"], case["key_heads"], case["dim"], rotary_dim=case["rotary"],
                               layout=case["layout"], norm=None if case["norm"] == "none" else case["norm"],
                               dtype=case["dtype"], frequencies=s["frequencies"], rotation_scale=s["turn"],
                               epsilon=EPS)
        if s["weights"] is not None:
            op.prepare(**s["weights"])
        return op
    from afhip import window

    return window.WindowAttention(case["heads"], case["key_heads"], case["dim"], left=case["left"],
                                  right=case["right"], sinks=case["sinks"], dtype=case["dtype"])


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(s: dict):
    kind = s["case"]["kind"]
    if own:
        op = s["op"]
        if kind == "rotary":
            if "k_cache" in s:
                q, k, v = op(s["q"], s["k"], s["v"], past=s["past"], lengths=s["lengths"], k_cache=s["k_cache"],
                             v_cache=s["v_cache"])
                return {"q": q, "k": k, "v": v}
            q, k = op(s["q"], s["k"], past=s["past"], lengths=s["lengths"])
            return {"q": q, "k": k}
        if kind == "rotary_backward":
            return op.backward(s["q"], s["k"], s["dq"], s["dk"], past=s["past"], lengths=s["lengths"])
        if kind == "attention":
            out, lse = op(s["q"], s["k"], s["v"], query_lengths=s["query_lengths"], key_lengths=s["key_lengths"],
                          return_lse=True)
            return {"out": out, "lse": lse}
        dq, dk, dv = op.backward(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"],
                                 query_lengths=s["query_lengths"], key_lengths=s["key_lengths"])
        return {"dq": dq, "dk": dk, "dv": dv}
    if kind == "rotary":
        return _turn(s)
    if kind == "rotary_backward":
        return _turn_back(s)
    if kind == "attention":
        out, lse = _attend(s)
        return {"out": out, "lse": lse}
    return _attend_back(s)


# The plain forms: 32 bits (positions' angles 64), rounded once at the end.

def _angles(s: dict):
    """(cosines, sines) [batch][tokens][1][pairs], the factor on what is turned in them."""
    q = s["q"]
    pos = torch.arange(q.shape[1], device=q.device, dtype=torch.float64).expand(q.shape[0], -1)
    if s["past"] is not None:
        pos = pos + s["past"][:, None]
    a = pos[:, :, None, None] * s["frequencies"].to(q.device)
    return (a.cos() * s["turn"]).float(), (a.sin() * s["turn"]).float()


def _rotate(x, cos, sin, case):
    r = case["rotary"]
    if case["layout"] == "half":
        x0, x1 = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
    else:
        x0, x1 = x[..., :r:2], x[..., 1:r:2]
        turned = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _normed(x, case):
    """(x over its root mean square or standard deviation, the reciprocal of that)."""
    if case["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = 1 / ((x * x).mean(-1, keepdim=True) + EPS).sqrt()
    return x * r, r


def _live(s: dict):
    """Which tokens the sequences have, [batch][tokens]."""
    q = s["q"]
    at = torch.arange(q.shape[1], device=q.device)
    lengths = s["lengths"]
    return at < lengths[:, None] if lengths is not None else at.expand(q.shape[0], -1) >= 0


def _turn(s: dict):
    case = s["case"]
    cos, sin = _angles(s)
    live = _live(s)[:, :, None, None]
    out = {}
    for name, x, weights in (("q", s["q"], "query"), ("k", s["k"], "key")):
        y = x.float()
        if case["norm"] != "none":
            y = _normed(y, case)[0] * s["weights"][weights + "_scale"]
            if case["norm"] == "layer":
                y = y + s["weights"][weights + "_offset"]
        out[name] = torch.where(live, _rotate(y, cos, sin, case), 0.0).to(x.dtype)
    if "k_cache" in s:
        b, t = s["q"].shape[:2]
        row = torch.arange(t, device=s["q"].device).expand(b, -1)
        if s["past"] is not None:
            row = row + s["past"][:, None]
        entry = torch.arange(b, device=s["q"].device)[:, None].expand(-1, t)
        if s["lengths"] is not None:
            at = _live(s)
            entry, row = entry[at], row[at]
            s["k_cache"][entry, row], s["v_cache"][entry, row] = out["k"][at], s["v"][at]
        else:
            s["k_cache"][entry, row], s["v_cache"][entry, row] = out["k"], s["v"]
        out["k"], out["v"] = s["k_cache"], s["v_cache"]
    return out


def _turn_back(s: dict):
    case = s["case"]
    cos, sin = _angles(s)
    live = _live(s)[:, :, None, None]
    out = {}
    for name, x, dy, weights in (("q", s["q"], s["dq"], "query"), ("k", s["k"], s["dk"], "key")):
        g = _rotate(dy.float(), cos, -sin, case)
        if case["norm"] != "none":
            g = torch.where(live, g, 0.0)
            xhat, r = _normed(x.float(), case)
            # Sums over every token and head, long ones: in 64 bits.
            out["d" + weights + "_scale"] = (g * xhat).sum((0, 1, 2), dtype=torch.float64).float()
            if case["norm"] == "layer":
                out["d" + weights + "_offset"] = g.sum((0, 1, 2), dtype=torch.float64).float()
            g = g * s["weights"][weights + "_scale"]
            inner = g - xhat * (g * xhat).mean(-1, keepdim=True)
            if case["norm"] == "layer":
                inner = inner - g.mean(-1, keepdim=True)
            g = r * inner
        out["d" + name] = torch.where(live, g, 0.0).to(x.dtype)
    return out


def _grouped(x, key_heads: int):
    """[batch][tokens][heads][channels] -> [batch * key_heads][group * tokens][channels], 32 bits."""
    b, t, h, d = x.shape
    x = x.float().unflatten(2, (key_heads, h // key_heads)).permute(0, 2, 3, 1, 4)
    return x.reshape(b * key_heads, (h // key_heads) * t, d)


def _ungrouped(x, batch: int, tokens: int):
    """The way back from _grouped."""
    hk = x.shape[0] // batch
    x = x.reshape(batch, hk, -1, tokens, x.shape[-1]).permute(0, 3, 1, 2, 4)
    return x.flatten(2, 3)


def _visible(s: dict):
    """Which keys a query sees, [batch][1][1][queries][keys]."""
    case, q, k = s["case"], s["q"], s["k"]
    b, tq, tk = q.shape[0], q.shape[1], k.shape[1]
    i = torch.arange(tq, device=q.device)[None, :, None]
    j = torch.arange(tk, device=q.device)[None, None, :]
    ql = s["query_lengths"][:, None, None] if s["query_lengths"] is not None else tq
    kl = s["key_lengths"][:, None, None] if s["key_lengths"] is not None else tk
    p = i + (kl - ql)
    seen = (j < kl) & (i < ql)
    if case["right"] >= 0:
        seen = seen & (j <= p + case["right"])
    if case["left"] >= 0:
        seen = seen & ((j >= p - case["left"]) | (j < case["sinks"]))
    return seen.expand(b, tq, tk)[:, None, None]


def _scores(s: dict):
    """The scaled scores, -inf where nothing is seen, [batch * key_heads][group * queries][keys]."""
    case, q, k = s["case"], s["q"], s["k"]
    b, tq, hk, tk = q.shape[0], q.shape[1], case["key_heads"], k.shape[1]
    x = torch.matmul(_grouped(q, hk), _grouped(k, hk).transpose(1, 2)) * (1 / math.sqrt(case["dim"]))
    seen = _visible(s)
    return torch.where(seen, x.view(b, hk, -1, tq, tk), -math.inf).view(b * hk, -1, tk)


def _attend(s: dict):
    case, q = s["case"], s["q"]
    b, tq, hk = q.shape[0], q.shape[1], case["key_heads"]
    x = _scores(s)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    x = (x - top).exp()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x, _grouped(s["v"], hk)) / torch.where(total == 0, 1.0, total)
    lse = _ungrouped(top + total.log(), b, tq)
    return _ungrouped(out, b, tq).to(q.dtype).contiguous(), lse[..., 0].transpose(1, 2).contiguous()


def _attend_back(s: dict):
    case, q, k = s["case"], s["q"], s["k"]
    b, tq, tk, hk = q.shape[0], q.shape[1], k.shape[1], case["key_heads"]
    gq, gk, gv, gd = (_grouped(x, hk) for x in (q, k, s["v"], s["dout"]))
    x = _scores(s)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    x = (x - top).exp()
    total = x.sum(-1, keepdim=True)
    x = x / torch.where(total == 0, 1.0, total)
    dv = torch.matmul(x.transpose(1, 2), gd)
    g = torch.matmul(gd, gv.transpose(1, 2))
    g = x * (g - (g * x).sum(-1, keepdim=True)) * (1 / math.sqrt(case["dim"]))
    dq, dk = torch.matmul(g, gk), torch.matmul(g.transpose(1, 2), gq)
    dt = q.dtype
    return {"dq": _ungrouped(dq, b, tq).to(dt).contiguous(), "dk": _ungrouped(dk, b, tk).to(dt).contiguous(),
            "dv": _ungrouped(dv, b, tk).to(dt).contiguous()}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one sequence and head at a time
# ---------------------------------------------------------------------------

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return _exact_rotary(s) if case["kind"].startswith("rotary") else _exact_attention(s)


def _exact_rotary(s: dict):
    case = s["case"]
    r = case["rotary"]
    ql, kl = _lengths(case)
    back = case["kind"] == "rotary_backward"
    first = [2 * j if case["layout"] == "interleaved" else j for j in range(r // 2)]
    second = [2 * j + 1 if case["layout"] == "interleaved" else j + r // 2 for j in range(r // 2)]
    freq = s["frequencies"].to(s["q"].device)
    out = {}
    for name, weights in (("q", "query"), ("k", "key")):
        x = s[name].double()
        params = [w.double().requires_grad_(back) for w in
                  ((s["weights"][weights + "_scale"], s["weights"].get(weights + "_offset")) if s["weights"] else ())
                  if w is not None]
        result = torch.zeros_like(x)
        sums = [torch.zeros_like(w) for w in params]
        for b, n in enumerate(ql):
            v = x[b, :n].detach().requires_grad_(back)
            y = v
            if case["norm"] == "rms":
                y = v / (v.square().mean(-1, keepdim=True) + EPS).sqrt() * params[0]
            elif case["norm"] == "layer":
                y = (v - v.mean(-1, keepdim=True)) / (v.var(-1, unbiased=False, keepdim=True) + EPS).sqrt()
                y = y * params[0] + params[1]
            turn = torch.polar(torch.tensor(s["turn"], dtype=torch.float64, device=x.device),
                               (torch.arange(n, device=x.device, dtype=torch.float64) + (kl[b] - n))[:, None] * freq)
            z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
            y = y.clone()
            y[..., first], y[..., second] = z.real, z.imag
            if back:
                got = torch.autograd.grad(y, [v] + params, s["d" + name][b, :n].double())
                result[b, :n] = got[0]
                sums = [t + g for t, g in zip(sums, got[1:])]
            else:
                result[b, :n] = y
        if back:
            out["d" + name] = result
            for suffix, total in zip(("_scale", "_offset"), sums):
                out["d" + weights + suffix] = total
        else:
            out[name] = result
    if "k_cache" in s:
        k, v = s["k_cache"].double(), s["v_cache"].double()
        for b, n in enumerate(ql):
            k[b, kl[b] - n:kl[b]], v[b, kl[b] - n:kl[b]] = out["k"][b, :n], s["v"][b, :n].double()
        out["k"], out["v"] = k, v
    return out


def _exact_attention(s: dict):
    case = s["case"]
    back = case["kind"] == "attention_backward"
    group = case["heads"] // case["key_heads"]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    out, lse = torch.zeros_like(q), torch.full((q.shape[0], q.shape[2], q.shape[1]), -math.inf, dtype=torch.float64,
                                               device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b, (nq, nk) in enumerate(zip(*_lengths(case))):
        p = torch.arange(nk - nq, nk, device=q.device)[:, None]
        j = torch.arange(nk, device=q.device)[None]
        hidden = torch.zeros(nq, nk, dtype=torch.bool, device=q.device)
        if case["left"] >= 0:
            hidden |= (p - j > case["left"]) & (j >= case["sinks"])
        if case["right"] >= 0:
            hidden |= j - p > case["right"]
        for h in range(case["heads"]):
            a, c, d = (x.detach().requires_grad_(back) for x in
                       (q[b, :nq, h], k[b, :nk, h // group], v[b, :nk, h // group]))
            x = (a @ c.T / case["dim"] ** 0.5).masked_fill(hidden, -math.inf)
            y = torch.softmax(x, -1) @ d
            if back:
                g = torch.autograd.grad(y, (a, c, d), s["dout"][b, :nq, h].double())
                dq[b, :nq, h] = g[0]
                dk[b, :nk, h // group] += g[1]
                dv[b, :nk, h // group] += g[2]
            else:
                out[b, :nq, h] = y
                lse[b, h, :nq] = torch.logsumexp(x, -1)
    return {"dq": dq, "dk": dk, "dv": dv} if back else {"out": out, "lse": lse}
