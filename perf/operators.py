"""The operators of a rank's training and serving step that stand beside the collectives, as cases.

Four operators: the global gradient norm with clipping, layer / RMS norm with its gradients, the
embedding lookup with its gradient, and tokens sorted by expert and back with its gradients.
``run`` computes them in plain torch operations (32 bits, rounded once), or, where ``own`` is
true, through the package's entry points. ``exact`` computes the same outputs in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_EPS = 1e-5        # of the norms
_CLIP_EPS = 1e-6   # added to the gradient norm before the division


def _dtype(name):
    return getattr(torch, name)


def _bytes(name):
    return torch.empty(0, dtype=_dtype(name)).element_size()


# ---------------------------------------------------------------- cases
def listed():
    return [
        # Global gradient norm and clipping. The bias gradients of a data-parallel step: many tensors of 4 KiB.
        {"name": "clip_biases", "op": "clip", "vocab": 0, "hidden": 0, "intermediate": 0, "kv": 0, "layers": 0,
         "biases": 256, "bias": 1024, "dtype": "float32", "out": "float32", "clips": True},
        # A small model's gradients with vectors of odd length between the matrices; bf16 gradients clipped
        # into the optimizer's 32-bit ones.
        {"name": "clip_small_model", "op": "clip", "vocab": 1024, "hidden": 256, "intermediate": 768, "kv": 128,
         "layers": 8, "biases": 24, "bias": 771, "dtype": "bfloat16", "out": "float32", "clips": True},
        # The 8B shapes, embedding table and one layer, in a step whose norm is below the bound (most steps).
        {"name": "clip_idle_8b_layer", "op": "clip", "vocab": 128256, "hidden": 4096, "intermediate": 14336,
         "kv": 1024, "layers": 1, "biases": 0, "bias": 0, "dtype": "bfloat16", "out": "", "clips": False},
        # The 8B shapes, four layers without the table, in a step that is clipped.
        {"name": "clip_8b_layers", "op": "clip", "vocab": 0, "hidden": 4096, "intermediate": 14336, "kv": 1024,
         "layers": 4, "biases": 0, "bias": 0, "dtype": "bfloat16", "out": "bfloat16", "clips": True},
        # Norms. A decoding step of a few sequences.
        {"name": "norm_decode", "op": "norm", "kind": "rms", "rows": 4, "hidden": 4096, "dtype": "bfloat16",
         "weight": "bfloat16", "train": False},
        # A training step over the tensor-parallel MLP's activations: 8192 tokens of 8192.
        {"name": "norm_train_tokens", "op": "norm", "kind": "rms", "rows": 8192, "hidden": 8192, "dtype": "bfloat16",
         "weight": "bfloat16", "train": True},
        # Layer norm with 32-bit weights over rows of odd length (rows start at every alignment).
        {"name": "norm_train_odd", "op": "norm", "kind": "layer", "rows": 2051, "hidden": 1531, "dtype": "float16",
         "weight": "float32", "train": True},
        # Embedding. A decoding step of 64 sequences on the 8B table.
        {"name": "embed_decode", "op": "embedding", "ids": 64, "vocab": 128256, "hidden": 4096, "dtype": "bfloat16",
         "first": 0, "rows": 128256, "scale": 1.0, "padding": False, "train": False},
        # A training step of 32768 tokens on the 8B table: word frequencies, so a few tokens are everywhere.
        {"name": "embed_train_8b", "op": "embedding", "ids": 32768, "vocab": 128256, "hidden": 4096,
         "dtype": "bfloat16", "first": 0, "rows": 128256, "scale": 1.0, "padding": False, "train": True},
        # One rank's shard of a small 32-bit table: scaled, padded, most tokens on other ranks, odd sizes.
        {"name": "embed_train_shard", "op": "embedding", "ids": 3001, "vocab": 1024, "hidden": 251,
         "dtype": "float32", "first": 129, "rows": 511, "scale": 16.0, "padding": True, "train": True},
        # Experts. A decoding step.
        {"name": "experts_decode", "op": "experts", "tokens": 8, "top": 2, "experts": 8, "hidden": 4096,
         "dtype": "bfloat16", "weight": "float32", "drops": False, "train": False},
        # A training step: 8192 tokens, each to 8 of 64 experts.
        {"name": "experts_train", "op": "experts", "tokens": 8192, "top": 8, "experts": 64, "hidden": 4096,
         "dtype": "bfloat16", "weight": "float32", "drops": False, "train": True},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """Sizes spread over the listed ranges; no drawn case moves more bytes than its operator's largest listed one."""
    op = rng.choice(["clip", "norm", "embedding", "experts"])
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    if op == "clip":
        out = rng.choice(["", dtype, "float32"])
        hidden = _log_int(rng, 32, 4096)
        inter = _log_int(rng, hidden, 4 * hidden)
        kv = max(1, hidden // rng.choice([1, 2, 4, 8]))
        per_layer = 2 * hidden * hidden + 2 * kv * hidden + 3 * inter * hidden
        budget = 700_000_000 // (2 if dtype == "float32" or out == "float32" else 1)
        layers = _log_int(rng, 1, max(1, min(48, budget // (2 * per_layer))))
        vocab = rng.choice([0, _log_int(rng, 64, max(64, min(128256, budget // (2 * hidden))))])
        return {"op": op, "vocab": vocab, "hidden": hidden, "intermediate": inter, "kv": kv, "layers": layers,
                "biases": rng.choice([0, 1, _log_int(rng, 2, 256)]), "bias": _log_int(rng, 1, 4099), "dtype": dtype,
                "out": out, "clips": out != ""}
    if op == "norm":
        hidden = _log_int(rng, 8, 16384)
        if rng.random() < 0.7:
            hidden = max(8, hidden // 8 * 8)
        most = 8192 * 8192 // (2 if dtype == "float32" else 1)
        return {"op": op, "kind": rng.choice(["layer", "rms"]), "rows": _log_int(rng, 1, min(65536, most // hidden)),
                "hidden": hidden, "dtype": dtype, "weight": rng.choice([dtype, "float32"]),
                "train": rng.random() < 0.6}
    if op == "embedding":
        hidden = _log_int(rng, 8, 8192)
        if rng.random() < 0.7:
            hidden = max(8, hidden // 8 * 8)
        size = 4 if dtype == "float32" else 2
        vocab = _log_int(rng, 64, min(256000, 1_000_000_000 // (hidden * size)))
        rows = rng.choice([vocab, max(1, vocab // rng.choice([2, 4, 8]))])
        return {"op": op, "ids": _log_int(rng, 1, min(131072, 250_000_000 // (hidden * size))), "vocab": vocab,
                "hidden": hidden, "dtype": dtype, "first": rng.choice([0, vocab - rows]), "rows": rows,
                "scale": rng.choice([1.0, 0.5, math.sqrt(hidden)]), "padding": rng.random() < 0.3,
                "train": rng.random() < 0.6}
    hidden = _log_int(rng, 8, 8192)
    if rng.random() < 0.7:
        hidden = max(8, hidden // 8 * 8)
    experts = _log_int(rng, 1, 512)
    top = rng.randint(1, min(8, experts))
    size = 4 if dtype == "float32" else 2
    return {"op": op, "tokens": _log_int(rng, 1, min(131072, 400_000_000 // (hidden * size * top))), "top": top,
            "experts": experts, "hidden": hidden, "dtype": dtype, "weight": rng.choice([dtype, "float32"]),
            "drops": rng.random() < 0.3, "train": rng.random() < 0.6}


def _shapes(case):
    """The gradients' shapes: a table, then each layer's matrices and vectors, then bias vectors."""
    h, f, kv = case["hidden"], case["intermediate"], case["kv"]
    layer = [(h,), (h, h), (kv, h), (kv, h), (h, h), (h,), (f, h), (f, h), (h, f)]
    return ([(case["vocab"], h)] if case["vocab"] else []) + layer * case["layers"] + [(case["bias"],)] * case["biases"]


def _elements(case):
    return sum(math.prod(s) for s in _shapes(case))


def _views(case, flat):
    shapes = _shapes(case)
    return [part.view(s) for part, s in zip(torch.split(flat, [math.prod(s) for s in shapes]), shapes)]


# ---------------------------------------------------------------- inputs
def _zipf(ids, vocab, g):
    """Token ids with the frequencies of words: rank r about as often as 1 / (r + 2.7)."""
    weight = 1.0 / (torch.arange(vocab, device="cuda", dtype=torch.float64) + 2.7)
    total = torch.cumsum(weight, 0)
    u = torch.rand(ids, device="cuda", dtype=torch.float64, generator=g) * total[-1]
    return torch.searchsorted(total, u).clamp_(max=vocab - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, std=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * std).to(_dtype(dtype))

    st = dict(case)
    if case["op"] == "clip":
        # Gradients are views of one flat storage, as a data-parallel sync lays them out; so are the clipped ones.
        st["flat"] = normal((_elements(case),), case["dtype"], 1e-3)
        st["grads"] = _views(case, st["flat"])
        st["clipped"] = torch.empty_like(st["flat"], dtype=_dtype(case["out"])) if case["out"] else None
        st["outs"] = _views(case, st["clipped"]) if case["out"] else None
        # The norm is about 1e-3 sqrt(n): a bound below it clips, one above does not.
        st["max_norm"] = 1e-3 * math.sqrt(_elements(case)) * (0.3 if case["clips"] else 4.0)
    elif case["op"] == "norm":
        n, h = case["rows"], case["hidden"]
        wide = 1.0 + 9.0 * (torch.rand(h, device="cuda", generator=g) < 0.01)  # a few channels carry large values
        st["x"] = ((torch.randn(n, h, device="cuda", generator=g) + 0.3) * wide).to(_dtype(case["dtype"]))
        st["weight"] = (1.0 + 0.1 * torch.randn(h, device="cuda", generator=g)).to(_dtype(case["weight"]))
        st["bias"] = normal((h,), case["weight"], 0.1) if case["kind"] == "layer" else None
        if case["train"]:
            st["dy"] = normal((n, h), case["dtype"], 1e-2)
    elif case["op"] == "embedding":
        st["table"] = normal((case["rows"], case["hidden"]), case["dtype"], 0.02)
        st["ids"] = _zipf(case["ids"], case["vocab"], g)
        st["padding_idx"] = case["first"] + 1 if case["padding"] else None
        if case["padding"]:  # a padded batch: its tail is padding
            st["ids"][case["ids"] - case["ids"] // 8:] = st["padding_idx"]
        if case["train"]:
            st["dy"] = normal((case["ids"], case["hidden"]), case["dtype"], 1e-2)
    else:
        t, k, e, h = case["tokens"], case["top"], case["experts"], case["hidden"]
        lean = torch.randn(e, device="cuda", generator=g)  # some experts are chosen more often than others
        score = lean + 1.5 * torch.randn(t, e, device="cuda", generator=g)
        best = torch.topk(score, k, dim=1)
        st["ids"] = best.indices.to(torch.int32)
        if case["drops"]:
            st["ids"][torch.rand(t, k, device="cuda", generator=g) < 0.1] = -1
        st["weights"] = torch.softmax(best.values, 1).to(_dtype(case["weight"]))
        st["x"] = normal((t, h), case["dtype"])
        st["rows"] = normal((t * k, h), case["dtype"])       # what the experts answered
        if case["train"]:
            st["dy"] = normal((t, h), case["dtype"], 1e-2)
            st["dsorted"] = normal((t * k, h), case["dtype"], 1e-2)  # the gradient of the sorted rows
    return st


# ---------------------------------------------------------------- one pass
def run(st):
    if own:
        return _own(st)
    return {"clip": _plain_clip, "norm": _plain_norm, "embedding": _plain_embedding, "experts": _plain_experts}[st["op"]](st)


def _own(st):
    from originccl_b200.ops import embedding, experts, gradients, norm

    if st["op"] == "clip":
        total = gradients.clip_grad_norm(st["grads"], st["max_norm"], eps=_CLIP_EPS, outs=st["outs"])
        return total, st["flat"] if st["outs"] is None else st["clipped"]
    if st["op"] == "norm":
        x, w, b = st["x"], st["weight"], st["bias"]
        if st["kind"] == "layer":
            y, mean, rstd = norm.layer_norm_forward(x, w, b, eps=_EPS)
            if not st["train"]:
                return y, mean, rstd
            return (y, mean, rstd) + norm.layer_norm_backward(st["dy"], x, mean, rstd, w)
        y, rstd = norm.rms_norm_forward(x, w, eps=_EPS)
        if not st["train"]:
            return y, rstd
        return (y, rstd) + norm.rms_norm_backward(st["dy"], x, rstd, w)
    if st["op"] == "embedding":
        y = embedding.embedding_forward(st["ids"], st["table"], scale=st["scale"], first_row=st["first"])
        if not st["train"]:
            return y
        return y, embedding.embedding_backward(st["dy"], st["ids"], st["table"].shape[0], scale=st["scale"],
                                               first_row=st["first"], padding_idx=st["padding_idx"])
    order = experts.sort_by_expert(st["ids"], st["experts"])
    out = (order.slots, order.sources, order.offsets, experts.dispatch_forward(st["x"], order),
           experts.combine_forward(st["rows"], order, st["weights"]))
    if not st["train"]:
        return out
    drows, dweights = experts.combine_backward(st["dy"], st["rows"], order, st["weights"])
    return out + (drows, dweights, experts.dispatch_backward(st["dsorted"], order))


def _plain_clip(st):
    flat = torch.cat([t.reshape(-1) for t in st["grads"]]).float()
    total = (flat * flat).sum().sqrt()
    coef = torch.clamp(st["max_norm"] / (total + _CLIP_EPS), max=1.0)
    return total, (flat * coef).to((st["outs"] or st["grads"])[0].dtype)


def _plain_norm(st):
    x, w = st["x"].float(), st["weight"].float()
    if st["kind"] == "layer":
        mean = x.mean(1)
        xc = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((xc * xc).mean(1) + _EPS)
        xh = xc * rstd[:, None]
        out = ((xh * w + st["bias"].float()).to(st["x"].dtype), mean, rstd)
    else:
        rstd = 1.0 / torch.sqrt((x * x).mean(1) + _EPS)
        xh = x * rstd[:, None]
        out = ((xh * w).to(st["x"].dtype), rstd)
    if not st["train"]:
        return out
    dy = st["dy"].float()
    g = dy * w
    inner = g - xh * (g * xh).mean(1, keepdim=True)
    if st["kind"] == "layer":
        inner = inner - g.mean(1, keepdim=True)
    out += ((inner * rstd[:, None]).to(st["x"].dtype), (dy * xh).sum(0).to(st["weight"].dtype))
    if st["kind"] == "layer":
        out += (dy.sum(0).to(st["bias"].dtype),)
    return out


def _plain_embedding(st):
    table, row = st["table"], st["ids"] - st["first"]
    inside = (row >= 0) & (row < table.shape[0])
    row = torch.where(inside, row, 0)
    y = (table[row].float() * st["scale"] * inside[:, None]).to(table.dtype)
    if not st["train"]:
        return y
    if st["padding_idx"] is not None:
        inside = inside & (st["ids"] != st["padding_idx"])
    grad = torch.zeros(table.shape, device=table.device)
    grad.index_add_(0, row, st["dy"].float() * inside[:, None])
    return y, (grad * st["scale"]).to(table.dtype)


def _plain_experts(st):
    ids, (t, k), e = st["ids"], st["ids"].shape, st["experts"]
    key = torch.where((ids >= 0) & (ids < e), ids, e).reshape(-1)
    order = torch.sort(key, stable=True).indices
    counts = torch.zeros(e + 1, dtype=torch.int64, device=ids.device).index_add_(0, key.long(), torch.ones_like(order))
    offsets = torch.zeros(e + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = torch.cumsum(counts[:e], 0)
    place = torch.empty_like(order)
    place[order] = torch.arange(t * k, device=ids.device)
    kept = place < offsets[e]
    slots = torch.where(kept, place, -1).view(t, k).to(torch.int32)
    live = torch.arange(t * k, device=ids.device) < offsets[e]
    sources = torch.where(live, order, -1).to(torch.int32)
    sorted_rows = st["x"][order // k] * live[:, None]
    keep, at = kept.view(t, k), torch.where(kept, place, 0).view(t, k)
    w = st["weights"].float() * keep
    picked = st["rows"][at].float()
    y = (picked * w[..., None]).sum(1).to(st["x"].dtype)
    out = (slots, sources, offsets, sorted_rows, y)
    if not st["train"]:
        return out
    dy = st["dy"].float()
    drows = (dy[order // k] * (w.reshape(-1)[order] * live)[:, None]).to(st["x"].dtype)
    dweights = ((picked * dy[:, None, :]).sum(2) * keep).to(st["weights"].dtype)
    dx = (st["dsorted"][at].float() * keep[..., None]).sum(1).to(st["x"].dtype)
    return out + (drows, dweights, dx)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = _bytes(case["dtype"])
    if case["op"] == "clip":
        n = _elements(case)
        return {"bytes": n * (size + (_bytes(case["out"]) if case["out"] else 0)),
                "flops": (3 if case["clips"] else 2) * n}
    if case["op"] == "norm":
        n, h = case["rows"], case["hidden"]
        vectors = (2 if case["kind"] == "layer" else 1) * h * _bytes(case["weight"])
        moved, ops = 2 * n * h * size + 8 * n + vectors, 6 * n * h
        if case["train"]:  # dy in, dx and the weights' gradients out
            moved, ops = moved + 2 * n * h * size + vectors, ops + 12 * n * h
        return {"bytes": moved, "flops": ops}
    if case["op"] == "embedding":
        n, h = case["ids"], case["hidden"]
        # The distinct rows that n draws with the frequencies of words touch, about.
        total = math.log((case["vocab"] + 2.7) / 2.7)
        hit, step = 0.0, max(1, case["rows"] // 2048)
        for r in range(case["first"], case["first"] + case["rows"], step):
            hit += step * -math.expm1(-n / (total * (r + 2.7)))
        hit = min(hit, n, case["rows"])
        moved, ops = 8 * n + (hit + n) * h * size, n * h
        if case["train"]:
            moved, ops = moved + (n + case["rows"]) * h * size, ops + 2 * n * h
        return {"bytes": int(moved), "flops": ops}
    t, k, h = case["tokens"], case["top"], case["hidden"]
    moved = 4 * t * k + 8 * t * k + t * k * _bytes(case["weight"]) + 2 * (t + t * k) * h * size
    ops = 2 * t * k * h
    if case["train"]:
        moved, ops = moved + 2 * (t + t * k) * h * size + t * k * _bytes(case["weight"]), ops + 4 * t * k * h
    return {"bytes": moved, "flops": ops}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "clip":
        squares = [torch.linalg.vector_norm(t, dtype=f64) ** 2 for t in st["grads"]]
        total = torch.sqrt(torch.stack(squares).sum())
        coef = min(1.0, st["max_norm"] / (float(total) + _CLIP_EPS))
        return total, st["flat"].to(f64) * coef
    if case["op"] == "norm":
        return _exact_norm(st, f64)
    if case["op"] == "embedding":
        ids, table = st["ids"], st["table"]
        first, rows = case["first"], case["rows"]
        y = torch.zeros(case["ids"], case["hidden"], dtype=f64, device="cuda")
        here = torch.nonzero((ids >= first) & (ids < first + rows)).flatten()
        y[here] = table.index_select(0, ids[here] - first).to(f64) * case["scale"]
        if not case["train"]:
            return y
        if st["padding_idx"] is not None:
            here = here[ids[here] != st["padding_idx"]]
        grad = torch.zeros(rows, case["hidden"], dtype=f64, device="cuda")
        for part in torch.split(here, 8192):
            grad.index_put_((ids[part] - first,), st["dy"][part].to(f64) * case["scale"], accumulate=True)
        return y, grad
    return _exact_experts(st, f64)


def _exact_norm(st, f64):
    x, w = st["x"].to(f64), st["weight"].to(f64)
    h = x.shape[1]
    mean = x.sum(1) / h if st["kind"] == "layer" else torch.zeros(x.shape[0], dtype=f64, device=x.device)
    x = x.sub_(mean[:, None])
    rstd = (torch.einsum("nh,nh->n", x, x) / h + _EPS).rsqrt()
    x = x.mul_(rstd[:, None])
    y = x * w + (st["bias"].to(f64) if st["kind"] == "layer" else 0.0)
    out = (y, mean, rstd) if st["kind"] == "layer" else (y, rstd)
    if not st["train"]:
        return out
    dy = st["dy"].to(f64)
    dw, db = torch.einsum("nh,nh->h", dy, x), dy.sum(0)
    a = torch.einsum("nh,nh,h->n", dy, x, w) / h
    b = dy @ w / h if st["kind"] == "layer" else torch.zeros_like(a)
    dx = (dy * w - b[:, None] - x * a[:, None]) * rstd[:, None]
    return out + ((dx, dw, db) if st["kind"] == "layer" else (dx, dw))


def _exact_experts(st, f64):
    ids = st["ids"].cpu().tolist()
    t, k, e, h = st["tokens"], st["top"], st["experts"], st["hidden"]
    lists = [[] for _ in range(e)]
    for token, chosen in enumerate(ids):
        for j, expert in enumerate(chosen):
            if 0 <= expert < e:
                lists[expert].append(token * k + j)
    flat = [a for one in lists for a in one]
    ends = [0]
    for one in lists:
        ends.append(ends[-1] + len(one))
    kept = len(flat)
    order = torch.tensor(flat, dtype=torch.int64, device="cuda")
    sources = torch.full((t * k,), -1, dtype=torch.int32, device="cuda")
    sources[:kept] = order.to(torch.int32)
    slots = torch.full((t * k,), -1, dtype=torch.int32, device="cuda")
    slots[order] = torch.arange(kept, dtype=torch.int32, device="cuda")
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    token = torch.div(order, k, rounding_mode="floor")
    sorted_rows = torch.zeros(t * k, h, dtype=f64, device="cuda")
    sorted_rows[:kept] = st["x"].to(f64)[token]
    w = st["weights"].to(f64).reshape(-1)
    y = torch.zeros(t, h, dtype=f64, device="cuda")
    y.index_add_(0, token, st["rows"][:kept].to(f64) * w[order][:, None])
    out = (slots.view(t, k), sources, offsets, sorted_rows, y)
    if not st["train"]:
        return out
    dy = st["dy"].to(f64)
    drows = torch.zeros(t * k, h, dtype=f64, device="cuda")
    drows[:kept] = dy[token] * w[order][:, None]
    dweights = torch.zeros(t * k, dtype=f64, device="cuda")
    dweights[order] = torch.einsum("nh,nh->n", dy[token], st["rows"][:kept].to(f64))
    dx = torch.zeros(t, h, dtype=f64, device="cuda")
    dx.index_add_(0, token, st["dsorted"][:kept].to(f64))
    return out + (drows, dweights.view(t, k), dx)
