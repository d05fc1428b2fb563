"""Cases for the row-scaled int8 products, the products grouped by expert and
the 8-bit activation checkpoints: inputs, plain forms, 64-bit forms and work.

Five kinds of call:
  int8        linear_int8: rows quantised to int8 with a scale each, times int8 weights with a scale per channel
  int8_group  linear_int8_grouped: the same with one weight matrix per group of rows
  group       gemm_grouped: 16-bit rows times their group's weights
  train       linear_grouped forward and backward (y, dx, dw)
  act8        linear / linear_grouped with save="int8": the backward pass reads 8-bit copies of the inputs
"""
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one new token through a square projection: latency and the weights' bytes
        {"name": "int8 one token", "op": "int8", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "bias": False},
        # a decoding batch through an up-projection with a bias
        {"name": "int8 decode 48", "op": "int8", "m": 48, "n": 10240, "k": 4096, "dtype": "fp16", "bias": True},
        # a prompt of odd length into an odd number of channels
        {"name": "int8 prompt odd", "op": "int8", "m": 1777, "n": 4099, "k": 4096, "dtype": "bf16", "bias": True},
        # a long batched prompt: bound by the tensor cores
        {"name": "int8 largest", "op": "int8", "m": 16384, "n": 8192, "k": 8192, "dtype": "bf16", "bias": False},
        # sixteen tokens, eight experts each of sixty-four: most experts see one to three rows
        {"name": "int8 experts decode", "op": "int8_group", "e": 64, "m": 128, "pad": 0, "n": 2048, "k": 4096,
         "dtype": "bf16", "bias": False},
        # a few routed tokens in 16 bits, in a padded buffer
        {"name": "experts decode", "op": "group", "e": 32, "m": 24, "pad": 8, "n": 4096, "k": 2048, "dtype": "bf16",
         "layout": "nk"},
        # a prompt's routed tokens, weights stored K x N, a result in fp32
        {"name": "experts prompt fp32", "op": "group", "e": 8, "m": 4001, "pad": 95, "n": 1536, "k": 2048,
         "dtype": "fp16", "layout": "kn", "out": "fp32"},
        # a training step of small experts with odd row counts, some empty
        {"name": "experts train odd", "op": "train", "e": 24, "m": 2999, "pad": 73, "n": 1032, "k": 520,
         "dtype": "fp16"},
        # a training step of a full batch of routed tokens
        {"name": "experts train", "op": "train", "e": 16, "m": 16384, "pad": 0, "n": 4096, "k": 2048,
         "dtype": "bf16"},
        # a small layer trained with 8-bit checkpoints: launch bound
        {"name": "act8 small", "op": "act8", "e": 0, "m": 515, "pad": 0, "n": 1024, "k": 768, "dtype": "fp16"},
        # experts trained with 8-bit checkpoints, odd row counts
        {"name": "act8 experts", "op": "act8", "e": 16, "m": 8003, "pad": 189, "n": 2048, "k": 2048,
         "dtype": "bf16"},
        # a large layer trained with 8-bit checkpoints
        {"name": "act8 large", "op": "act8", "e": 0, "m": 8192, "pad": 0, "n": 8192, "k": 4096, "dtype": "bf16"},
    ]


MOST_FLOPS = 2.0 * 16384 * 8192 * 8192


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return int(min(hi, max(step, step * round(v / step))))


def draw(rng):
    op = rng.choice(["int8", "int8", "int8_group", "group", "train", "act8"])
    while True:
        if op == "int8":
            case = {"op": op, "m": _log(rng, 1, 16384), "n": _log(rng, 96, 10240), "k": _log(rng, 128, 8192, 16),
                    "dtype": rng.choice(["bf16", "fp16", "fp32"]), "bias": rng.random() < 0.5}
        elif op == "int8_group":
            case = {"op": op, "e": rng.randint(2, 64), "m": _log(rng, 4, 8192), "pad": rng.choice([0, 0, 1, 37]),
                    "n": _log(rng, 256, 4096), "k": _log(rng, 256, 4096, 16), "dtype": rng.choice(["bf16", "fp16"]),
                    "bias": rng.random() < 0.5}
        elif op == "group":
            case = {"op": op, "e": rng.randint(2, 64), "m": _log(rng, 4, 16384), "pad": rng.choice([0, 0, 1, 37]),
                    "n": _log(rng, 256, 4096, 8), "k": _log(rng, 256, 4096, 8), "dtype": rng.choice(["bf16", "fp16"]),
                    "layout": rng.choice(["nk", "kn"])}
            if rng.random() < 0.3:
                case["out"] = "fp32"
        elif op == "train":
            case = {"op": op, "e": rng.randint(2, 32), "m": _log(rng, 64, 16384), "pad": rng.choice([0, 0, 1, 37]),
                    "n": _log(rng, 256, 4096, 8), "k": _log(rng, 256, 2048, 8), "dtype": rng.choice(["bf16", "fp16"])}
        else:
            e = rng.choice([0, 0, rng.randint(2, 24)])
            case = {"op": op, "e": e, "m": _log(rng, 64, 8192), "pad": rng.choice([0, 1, 37]) if e else 0,
                    "n": _log(rng, 256, 8192 if e == 0 else 2048, 8), "k": _log(rng, 256, 4096 if e == 0 else 2048, 16),
                    "dtype": rng.choice(["bf16", "fp16"])}
        if work(case)["flops"] <= MOST_FLOPS:
            return case


def _counts(case, seed):
    """Rows of each group: uneven, a few groups empty, summing to m."""
    r = random.Random(seed * 1000003 + 17)
    e, m = case["e"], case["m"]
    if not e:
        return [m]
    weight = [0.0 if r.random() < 0.1 else r.gammavariate(2.0, 1.0) for _ in range(e)]
    if not any(weight):
        weight[r.randrange(e)] = 1.0
    if m <= 4 * e:  # few rows: each goes to a group by itself
        picks = r.choices(range(e), weights=weight, k=m)
        return [picks.count(i) for i in range(e)]
    total, edge, edges = sum(weight), 0.0, []
    for w in weight:
        edge += w / total
        edges.append(min(m, round(edge * m)))
    edges[-1] = m
    return [b - a for a, b in zip([0] + edges, edges)]


def _activations(g, rows, k, dtype):
    """Normal values, a few channels larger (as activations have them), rows of different size."""
    x = torch.randn(rows, k, generator=g, device=DEV)
    x *= 1.0 + 7.0 * (torch.rand(1, k, generator=g, device=DEV) < 0.01)
    x *= 0.25 + torch.rand(rows, 1, generator=g, device=DEV)
    return x.to(dtype)


def _channel_codes(w):
    """int8 weights and their scales, one per output channel (the last axis is K)."""
    s = w.abs().amax(-1) / 127
    return torch.round(w / s[..., None]).clamp_(-127, 127).to(torch.int8), s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    op, n, k, dtype = case["op"], case["n"], case["k"], TYPES[case["dtype"]]
    rows = case["m"] + case.get("pad", 0)
    s = {"op": op, "rows": rows, "out": TYPES[case["out"]] if "out" in case else dtype}
    s["x"] = _activations(g, rows, k, dtype)
    e = case.get("e", 0)
    if e:
        counts = _counts(case, int(seed))
        edges = [0]
        for c in counts:
            edges.append(edges[-1] + c)
        s["offsets"] = torch.tensor(edges, dtype=torch.int32, device=DEV)
        s["most"] = max(counts)
    if op in ("int8", "int8_group"):
        w = torch.randn(*((e, n, k) if e else (n, k)), generator=g, device=DEV) * k ** -0.5
        s["w"], s["sw"] = _channel_codes(w)
        s["bias"] = torch.randn(*s["sw"].shape, generator=g, device=DEV) if case["bias"] else None
    else:
        s["layout"] = case.get("layout", "nk")
        shape = (n, k) if s["layout"] == "nk" else (k, n)
        s["w"] = (torch.randn(*((e,) + shape if e else shape), generator=g, device=DEV) * k ** -0.5).to(dtype)
    if op in ("train", "act8"):
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
        s["dy"] = (torch.randn(rows, n, generator=g, device=DEV) * n ** -0.5).to(dtype)
    return s


# ------------------------------------------------------------- plain forms --

def _quantize(x):
    """Codes and scales of each row, every step in fp32 (dividing by tensors: IEEE quotients)."""
    x = x.float()
    scale = x.abs().amax(-1) / torch.full((), 127.0, device=x.device)
    inv = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    q = (x * inv[..., None]).clamp(-127, 127)
    return torch.where(q >= 0, torch.floor(q + 0.5), torch.ceil(q - 0.5)), scale


class _Groups:
    """Rows laid out as one padded block per group, and back; rows behind the last group give zeros."""

    def __init__(self, offsets, most, rows):
        start, end = offsets[:-1].long(), offsets[1:].long()
        at = start[:, None] + torch.arange(most, device=offsets.device)
        self.inside = (at < end[:, None])[..., None]
        self.at = at.clamp(max=rows - 1)
        r = torch.arange(rows, device=offsets.device)
        self.group = (torch.searchsorted(offsets[1:].long(), r, right=True)).clamp(max=offsets.numel() - 2)
        self.place = (r - start[self.group]).clamp(max=most - 1)
        self.used = (r < end[-1])[:, None]

    def split(self, x):
        return torch.where(self.inside, x.float()[self.at], 0.0)

    def join(self, blocks):
        return torch.where(self.used, blocks[self.group, self.place], 0.0)


def _plain(s):
    op, x, w, out = s["op"], s["x"], s["w"], s["out"]
    groups = _Groups(s["offsets"], s["most"], s["rows"]) if "offsets" in s else None
    if op == "int8":
        codes, scale = _quantize(x)
        y = (codes @ w.float().t()) * scale[:, None] * s["sw"]
        return (y if s["bias"] is None else y + s["bias"]).to(out)
    if op == "int8_group":
        codes, scale = _quantize(x)
        y = (groups.split(codes) @ w.float().transpose(1, 2)) * s["sw"][:, None, :] * groups.split(scale[:, None])
        return groups.join(y if s["bias"] is None else y + s["bias"][:, None, :]).to(out)
    if op == "group":
        wf = w.float()
        return groups.join(groups.split(x) @ (wf.transpose(1, 2) if s["layout"] == "nk" else wf)).to(out)
    dy, kept = s["dy"], x.float()
    if op == "act8":
        codes, scale = _quantize(x)
        kept = codes * scale[:, None]
    wf = w.float()
    if groups is None:
        return {"y": (x.float() @ wf.t()).to(out), "dx": (dy.float() @ wf).to(out), "dw": (dy.float().t() @ kept).to(out)}
    gy = groups.split(dy)
    return {"y": groups.join(groups.split(x) @ wf.transpose(1, 2)).to(out), "dx": groups.join(gy @ wf).to(out),
            "dw": (gy.transpose(1, 2) @ groups.split(kept)).to(out)}


def run(state):
    s = state
    if not own:
        with torch.no_grad():
            return _plain(s)
    import tensorcoreptx_b200 as T
    if s["op"] == "int8":
        return T.linear_int8(s["x"], s["w"], s["sw"], s["bias"])
    if s["op"] == "int8_group":
        return T.linear_int8_grouped(s["x"], s["w"], s["offsets"], s["sw"], s["bias"])
    if s["op"] == "group":
        return T.gemm_grouped(s["x"], s["w"], s["offsets"], b_layout=s["layout"], out_dtype=s["out"])
    save = "int8" if s["op"] == "act8" else "input"
    if "offsets" in s:
        y = T.linear_grouped(s["x"], s["w"], s["offsets"], save=save)
    else:
        y = T.linear(s["x"], s["w"], save=save)
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw}


def work(case):
    m, n, k, e = case["m"], case["n"], case["k"], max(1, case.get("e", 0))
    el = 4 if case["dtype"] == "fp32" else 2
    used = min(e, m)  # groups that can have rows
    if case["op"] in ("int8", "int8_group"):
        return {"bytes": m * k * el + used * n * (k + 4 + (4 if case["bias"] else 0)) + m * n * el,
                "flops": 2.0 * m * n * k}
    if case["op"] == "group":
        return {"bytes": 2 * (m * k + used * n * k) + m * n * (4 if "out" in case else 2), "flops": 2.0 * m * n * k}
    # a training step: x, w and dy read, y, dx and dw written
    return {"bytes": 2 * (2 * m * k + 2 * m * n + 2 * e * n * k), "flops": 6.0 * m * n * k}


# ------------------------------------------------------------------ 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        x, w = s["x"].double(), s["w"].double()
        edges = s["offsets"].tolist() if "offsets" in s else [0, s["rows"]]
        w = w if "offsets" in s else w[None]
        per_group = []
        if case["op"] in ("int8", "int8_group", "act8"):
            top = x.abs().max(dim=1, keepdim=True).values
            t = x * 127 / torch.where(top > 0, top, torch.ones_like(top))
            x8 = torch.sign(t) * torch.floor(t.abs() + 0.5) * (top / 127)
        if case["op"] in ("int8", "int8_group"):
            sw = s["sw"].double().reshape(len(edges) - 1, -1)
            y = torch.zeros(s["rows"], case["n"], dtype=torch.float64, device=DEV)
            for i, (a, b) in enumerate(zip(edges, edges[1:])):
                y[a:b] = x8[a:b] @ (w[i] * sw[i][:, None]).t()
                if s["bias"] is not None:
                    y[a:b] += s["bias"].double().reshape(len(edges) - 1, -1)[i]
            return y
        if s["layout"] == "kn":
            w = w.transpose(1, 2)
        y = torch.zeros(s["rows"], case["n"], dtype=torch.float64, device=DEV)
        dx = torch.zeros_like(x)
        for i, (a, b) in enumerate(zip(edges, edges[1:])):
            y[a:b] = x[a:b] @ w[i].t()
            if "dy" in s:
                dx[a:b] = s["dy"][a:b].double() @ w[i]
                per_group.append(s["dy"][a:b].double().t() @ (x8 if case["op"] == "act8" else x)[a:b])
        if "dy" not in s:
            return y
        dw = torch.stack(per_group)
        return {"y": y, "dx": dx, "dw": dw if "offsets" in s else dw[0]}
