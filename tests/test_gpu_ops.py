"""The compute operators (gradient norm and clipping, norms, embedding, experts) on a GPU against
plain formulas in 64 bits.

Tolerances count roundings. An output is rounded once to its type: at most half a step,
``finfo(type).eps / 2`` of the value (plus half the smallest subnormal). Before that, 32-bit
arithmetic: a sum of m terms in any order is off by at most ``m * 2^-24`` times the sum of the terms'
magnitudes, each further operation by 2^-24 of its result. Each test says which m its kernel has.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids_of = lambda t: str(t).split(".")[-1]  # noqa: E731


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def check(got, exact, slack, what=""):
    """got is exact (64 bits) up to its type's rounding and ``slack`` before it."""
    assert got.shape == exact.shape, (what, got.shape, exact.shape)
    limit = (exact.abs() + slack) * (torch.finfo(got.dtype).eps / 2) + slack + TINY[got.dtype]
    off = (got.double() - exact).abs()
    bad = ~(off <= limit)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(off / limit).max().item():.3g} x the limit"


def randn(shape, dtype, seed, std=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std + mean).to(dtype)


# ---------------------------------------------------------------- norms
def norm64(kind, x, w, b, eps):
    x = x.double()
    mean = x.mean(-1) if kind == "layer" else torch.zeros(x.shape[:-1], dtype=torch.float64, device=x.device)
    xc = x - mean[..., None]
    rstd = (xc.square().mean(-1) + eps).rsqrt()
    xh = xc * rstd[..., None]
    y = xh if w is None else xh * w.double()
    return (y if b is None else y + b.double()), mean, rstd, xh


def check_norm(kind, x, w, b, eps, dy):
    """Forward and backward of one input. m = 64: a thread adds at most 32 elements (long rows: 40 at
    the tested lengths) and a block's tree 10; the rest is for the operations around the sums."""
    from originccl_b200.ops import norm
    m = 64 * U
    x2, dy2 = x.double(), dy.double()
    y64, mean64, rstd64, xh = norm64(kind, x, w, b, eps)
    layer = kind == "layer"
    if layer:
        y, mean, rstd = norm.layer_norm_forward(x, w, b, eps)
    else:
        y, rstd = norm.rms_norm_forward(x, w, eps)
    size = x2.abs().mean(-1, keepdim=True) * rstd64[..., None] if layer else torch.zeros_like(x2[..., :1])
    wa = 1.0 if w is None else w.double().abs()
    dxh = m * (xh.abs() + size)  # how far the normalised input may be off
    check(y, y64, dxh * wa + (0.0 if b is None else 2 * U * b.double().abs()), "y")
    if layer:
        check(mean, mean64, m * x2.abs().mean(-1), "mean")
    check(rstd, rstd64, m * rstd64 * (1 + size[..., 0] ** 2 * U), "rstd")

    if layer:
        dx, dw, db = norm.layer_norm_backward(dy, x, mean, rstd, w)
    else:
        dx, dw = norm.rms_norm_backward(dy, x, rstd, w)
        db = None
    g = dy2 if w is None else dy2 * w.double()
    m1 = g.mean(-1, keepdim=True) if layer else torch.zeros_like(g[..., :1])
    m2 = (g * xh).mean(-1, keepdim=True)
    r = rstd64[..., None]
    dm2 = (g.abs() * (dxh + m * xh.abs())).mean(-1, keepdim=True)
    dx64 = r * (g - m1 - xh * m2)
    slack = r * (m * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * m2.abs()) + xh.abs() * dm2 + dxh * m2.abs())
    check(dx, dx64, slack * 2, "dx")
    if w is None:
        assert dw is None and db is None
        return
    flat = (lambda t: t.reshape(-1, x.shape[-1]))
    rows = flat(x).shape[0]
    n = (rows / 148 + 64) * U  # a thread's rows, then at most 592 partial rows by 32 threads and a warp
    check(dw, flat(dy2 * xh).sum(0), n * flat(dy2 * xh).abs().sum(0) + flat(dy2.abs() * dxh).sum(0), "dw")
    if layer:
        check(db, flat(dy2).sum(0), n * flat(dy2).abs().sum(0), "db")


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("rows,h", [(1, 1), (3, 7), (1, 8), (5, 64), (17, 256), (9, 500), (33, 1000), (7, 1024), (300, 1531),
                                    (5, 2052), (1025, 4096), (6, 8192), (4, 8200), (5, 8201), (3, 16384), (2, 16386),
                                    (2, 40000), (2000, 33)])
def test_norms(kind, dtype, rows, h):
    for wtype in {dtype, torch.float32}:
        w, b = randn(h, wtype, 1, 0.2, 1.0), randn(h, wtype, 2, 0.3)
        x = randn((rows, h), dtype, 3, 2.0, 0.5)
        check_norm(kind, x, w, b if kind == "layer" else None, 1e-5, randn((rows, h), dtype, 4, 0.1))


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("h", [96, 101, 2048, 9000])
def test_norm_layouts(kind, h):
    """Rows apart, misaligned starts, leading dimensions, expanded gradients, no weight or bias."""
    w, b = randn(h, torch.bfloat16, 1, 0.2, 1.0), randn(h, torch.bfloat16, 2)
    wide = randn((13, h + 24), torch.bfloat16, 3)
    bias = b if kind == "layer" else None
    for x in (wide[:, :h], wide[:, 8:h + 8], wide[:, 3:h + 3], wide[::2, 1:h + 1], wide[:12, :h].reshape(3, 4, h),
              wide.t()[:h].t(), wide[:1, 5:h + 5].expand(6, h)):
        check_norm(kind, x, w, bias, 1e-6, randn(x.shape, torch.bfloat16, 5))
    x = wide[:, :h]
    check_norm(kind, x, w, bias, 1e-6, randn((1, h), torch.bfloat16, 6).expand(13, h))  # broadcast gradient
    check_norm(kind, x, w, bias, 1e-6, torch.full((1, 1), 0.5, device="cuda", dtype=torch.bfloat16).expand(13, h))
    check_norm(kind, x, None, None, 1e-6, randn(x.shape, torch.bfloat16, 7))
    if kind == "layer":
        check_norm(kind, x, w, None, 1e-6, randn(x.shape, torch.bfloat16, 8))
    whole = randn(h + 1, torch.bfloat16, 9, 0.2, 1.0)
    check_norm(kind, wide[:, :h], whole[1:], None, 1e-6, randn(x.shape, torch.bfloat16, 10))  # misaligned weight


def test_norm_of_large_offsets_and_equal_rows():
    """A mean far above the spread: the variance is of distances from the mean. Equal elements: zeros."""
    x = randn((8, 512), torch.float32, 1, 1.0, 1000.0)
    check_norm("layer", x, randn(512, torch.float32, 2, 0.1, 1.0), None, 1e-5, randn((8, 512), torch.float32, 3))
    from originccl_b200.ops import norm
    flat = torch.full((4, 320), 3.0, device="cuda", dtype=torch.bfloat16)
    y, mean, rstd = norm.layer_norm_forward(flat, None, None, 1e-5)
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(mean, torch.full_like(mean, 3.0))
    check(rstd, torch.full((4,), 1e-5, dtype=torch.float64, device="cuda").rsqrt(), 400 * U)


def test_norm_of_nothing_and_of_bad_values():
    from originccl_b200.ops import norm
    x = torch.empty(0, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    y, mean, rstd = norm.layer_norm_forward(x, w, w)
    dx, dw, db = norm.layer_norm_backward(x, x, mean, rstd, w)
    assert y.shape == dx.shape == (0, 16) and dw.eq(0).all() and db.eq(0).all()
    # A bad row stays in its row.
    x = randn((6, 300), torch.float32, 1)
    good, _ = norm.rms_norm_forward(x)
    x[2, 7], x[4, 0] = float("inf"), float("nan")
    y, _ = norm.rms_norm_forward(x)
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], good[keep]) and y[2, 7].isnan() and y[4].isnan().all()


def test_norm_in_place_and_into_a_strided_output():
    from originccl_b200.ops import norm
    x, w = randn((40, 640), torch.bfloat16, 1), randn(640, torch.bfloat16, 2)
    y, _ = norm.rms_norm_forward(x, w)
    wide = torch.full((40, 700), 7.0, device="cuda", dtype=torch.bfloat16)
    norm.rms_norm_forward(x, w, out=wide[:, 30:670])
    assert torch.equal(wide[:, 30:670], y) and wide[:, :30].eq(7).all() and wide[:, 670:].eq(7).all()
    inplace = x.clone()
    assert norm.rms_norm_forward(inplace, w, out=inplace)[0] is inplace and torch.equal(inplace, y)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norm_gradients_against_differences(kind):
    """d/ds of L(x + s v) in 64 bits by central differences (error s^2: below 1e-7 of the terms) against
    the kernels' gradients through autograd."""
    from originccl_b200.ops import norm
    x, v = randn((5, 1200), torch.float32, 1), randn((5, 1200), torch.float64, 2)
    w, b, t = randn(1200, torch.float32, 3, 0.2, 1.0), randn(1200, torch.float32, 4), randn((5, 1200), torch.float64, 5)
    xs, ws, bs = (p.clone().requires_grad_() for p in (x, w, b))
    y = norm.layer_norm(xs, ws, bs) if kind == "layer" else norm.rms_norm(xs, ws)
    (y.double() * t).sum().backward()
    f = lambda x, w, b: (norm64(kind, x, w, b if kind == "layer" else None, 1e-5)[0] * t).sum()  # noqa: E731
    s = 1e-4
    for p, grad, dirs in ((0, xs.grad, v), (1, ws.grad, v[0]), (2, bs.grad, v[1])):
        if p == 2 and kind == "rms":
            continue
        args = [x.double(), w.double(), b.double()]
        hi, lo = list(args), list(args)
        hi[p], lo[p] = args[p] + s * dirs, args[p] - s * dirs
        diff = (f(*hi) - f(*lo)) / (2 * s)
        terms = (grad.double() * dirs).abs().sum()
        assert abs((grad.double() * dirs).sum() - diff) <= 1e-5 * terms  # 128 x 2^-24 per term, and the difference's own


# ---------------------------------------------------------------- embedding
def table64(dy, ids, rows, scale, first, skip):
    d, i = dy.reshape(-1, dy.shape[-1]).double(), ids.reshape(-1).long()
    keep = (i >= first) & (i - first < rows) & ((i != skip) if skip is not None else True)
    out = torch.zeros(rows, d.shape[1], dtype=torch.float64, device=d.device)
    size, count = out.clone(), torch.zeros(rows, 1, dtype=torch.float64, device=d.device)
    out.index_add_(0, i[keep] - first, d[keep])
    size.index_add_(0, i[keep] - first, d[keep].abs())
    count.index_add_(0, i[keep] - first, torch.ones_like(d[keep][:, :1]))
    return out * scale, size * abs(scale), count


def some_ids(n, vocab, kind, seed, dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "same":
        return torch.full((n,), vocab // 2, device="cuda", dtype=dtype)
    if kind == "far":  # every value a 64-bit id may have
        ids = torch.randint(-vocab, 2 * vocab, (n,), device="cuda", generator=g)
        if dtype == torch.int64:
            ids[::7], ids[1::7] = 2 ** 63 - 1, -2 ** 63
        return ids.to(dtype)
    u = torch.rand(n, device="cuda", generator=g)
    return (vocab * (u ** 4 if kind == "skewed" else u)).long().clamp(max=vocab - 1).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("n,vocab,h,kind", [
    (1, 1, 1, "flat"), (1, 70000, 8, "flat"), (5, 3, 33, "flat"), (64, 1024, 256, "flat"), (777, 1023, 250, "skewed"),
    (4096, 1024, 64, "skewed"), (4097, 1025, 40, "skewed"), (9000, 128256, 16, "skewed"), (20000, 50, 24, "same"),
    (70001, 300, 9, "skewed"), (3000, 2000, 264, "far"), (300, 1100000, 8, "skewed"), (2049, 600, 3000, "skewed"),
    (16, 10, 2 ** 15 + 8, "flat"), (32768, 3000, 8, "skewed"), (32769, 1 << 21, 8, "flat"), (300001, 70000, 4, "far")])
def test_embedding(dtype, n, vocab, h, kind):
    from originccl_b200.ops import embedding
    for itype in (torch.int64, torch.int32):
        ids = some_ids(n, vocab, kind, 1, itype)
        w = randn((vocab, h), dtype, 2)
        inside = (ids >= 0) & (ids < vocab)
        for scale in (1.0, 1.7):
            y = embedding.embedding_forward(ids, w, scale)
            exact = w[torch.where(inside, ids, 0).long()].double() * scale * inside[:, None]
            check(y, exact, U * 2 * exact.abs(), "lookup")  # the scale itself is rounded to 32 bits
        dy = randn((n, h), dtype, 3)
        for skip in (None, vocab // 2):
            exact, size, count = table64(dy, ids, vocab, 0.7, 0, skip)
            got = embedding.embedding_backward(dy, ids, vocab, 0.7, padding_idx=skip)
            check(got, exact, (count + 2) * U * size, "gradient")
            assert got[count[:, 0] == 0].eq(0).all()
            again = embedding.embedding_backward(dy, ids, vocab, 0.7, padding_idx=skip)
            assert torch.equal(got.view(torch.uint8), again.view(torch.uint8)), "the same bits on every run"


@pytest.mark.parametrize("h", [48, 51])
def test_embedding_shards_add_up(h):
    """The shards of a table: outside ids give zeros, and rows and gradients come together."""
    from originccl_b200.ops import embedding
    w, ids = randn((1000, h), torch.bfloat16, 1), some_ids(500, 1000, "skewed", 2)
    whole = embedding.embedding_forward(ids, w, 2.0)
    dy = randn((500, h), torch.bfloat16, 3)
    grad = embedding.embedding_backward(dy, ids, 1000, 2.0, padding_idx=700)
    total, parts = torch.zeros_like(whole), []
    for first, rows in ((0, 1), (1, 332), (333, 667)):
        total += embedding.embedding_forward(ids, w[first:first + rows], 2.0, first_row=first)
        parts.append(embedding.embedding_backward(dy, ids, rows, 2.0, first_row=first, padding_idx=700))
    assert torch.equal(total, whole)
    # A shard's window edges lie elsewhere, so its sums may differ in their last bits.
    exact, size, count = table64(dy, ids, 1000, 2.0, 0, 700)
    check(torch.cat(parts), exact, (count + 2) * U * size)
    check(grad, exact, (count + 2) * U * size)


@pytest.mark.parametrize("otype", [torch.bfloat16, torch.float32], ids=ids_of)
@pytest.mark.parametrize("h", [64, 63])
def test_embedding_gradient_into_existing_storage(otype, h):
    from originccl_b200.ops import embedding
    n, vocab = 3000, 400
    ids = some_ids(n, vocab, "skewed", 1).reshape(30, 100)
    ids[:, 90:] = vocab + 5
    dy = randn((30, 100, h), torch.bfloat16, 2)
    dy[:, 90:] = float("nan")  # gradients of tokens of other shards are not read
    out = randn((vocab + 2, h), otype, 3)
    before, main = out.clone(), out[1:-1]
    exact, size, count = table64(torch.nan_to_num(dy), ids, vocab, 0.5, 0, None)
    got = embedding.embedding_backward(dy, ids, vocab, 0.5, out=main, accumulate=True)
    assert got is main
    old = before[1:-1].double()
    check(main, old + exact, (count + 3) * U * size + U * old.abs())
    gone = count[:, 0] == 0
    assert torch.equal(main[gone], before[1:-1][gone])
    assert torch.equal(out[0], before[0]) and torch.equal(out[-1], before[-1])  # neighbours stay
    embedding.embedding_backward(dy, ids, vocab, 0.5, out=main)
    check(main, exact, (count + 2) * U * size)
    assert main[gone].eq(0).all() and torch.equal(out[0], before[0]) and torch.equal(out[-1], before[-1])


def test_embedding_of_nothing_and_layouts():
    from originccl_b200.ops import embedding
    w = randn((50, 40), torch.float32, 1)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert embedding.embedding_forward(none, w).shape == (0, 40)
    assert embedding.embedding_backward(torch.empty(0, 40, device="cuda"), none, 50).eq(0).all()
    out = torch.ones(50, 40, device="cuda")
    embedding.embedding_backward(torch.empty(0, 40, device="cuda"), none, 50, out=out, accumulate=True)
    assert out.eq(1).all()
    ids = torch.arange(12, device="cuda").reshape(3, 4)
    assert embedding.embedding_forward(ids, torch.empty(0, 8, device="cuda")).eq(0).all()
    assert embedding.embedding_backward(randn((3, 4, 8), torch.float32, 2), ids, 0).shape == (0, 8)
    # strided tables, ids, gradients and outputs
    assert torch.equal(embedding.embedding_forward(ids.t(), w[:, 4:36]), w[:, 4:36][ids.t()])
    assert torch.equal(embedding.embedding_forward(ids, w.t()[:30].t()), w[:, :30][ids])
    dst = torch.zeros(12, 100, device="cuda")
    embedding.embedding_forward(ids.reshape(-1), w, out=dst[:, 7:47])
    assert torch.equal(dst[:, 7:47], w[:12]) and dst[:, :7].eq(0).all() and dst[:, 47:].eq(0).all()
    wide = randn((12, 90), torch.float32, 3)
    for dy in (wide[:, 11:51], wide[:1, :40].expand(12, 40)):
        got = embedding.embedding_backward(dy, ids.reshape(-1) // 2, 50)
        exact, size, count = table64(dy, ids.reshape(-1) // 2, 50, 1.0, 0, None)
        check(got, exact, (count + 2) * U * size)


def test_embedding_gradient_against_differences():
    """The lookup is linear: L(w + v) - L(w) in 64 bits is the gradient's product with v."""
    from originccl_b200.ops import embedding
    ids = some_ids(300, 90, "skewed", 1)
    w, v, t = randn((90, 70), torch.float32, 2), randn((90, 70), torch.float64, 3), randn((300, 70), torch.float32, 4)
    ws = w.clone().requires_grad_()
    (embedding.embedding(ids, ws, scale=3.0) * t).sum().backward()
    f = lambda w: (w[ids] * 3.0 * t.double()).sum()  # noqa: E731
    want = f(w.double() + v) - f(w.double())
    assert abs((ws.grad.double() * v).sum() - want) <= 302 * U * (ws.grad.double() * v).abs().sum() + 300 * 70 * U


# ---------------------------------------------------------------- experts
def order64(ids, experts):
    """slots, sources, offsets by a stable sort on the host."""
    flat = ids.reshape(-1).tolist()
    kept = sorted((e, a) for a, e in enumerate(flat) if 0 <= e < experts)
    slots, sources = [-1] * len(flat), [-1] * len(flat)
    for s, (_, a) in enumerate(kept):
        slots[a], sources[s] = s, a
    offsets = [sum(1 for e, _ in kept if e < i) for i in range(experts + 1)] if experts < 40 else None
    return slots, sources, offsets, len(kept)


@pytest.mark.parametrize("tokens,top,experts,kind", [
    (1, 1, 1, "flat"), (8, 2, 8, "flat"), (33, 3, 7, "far"), (1000, 1, 5, "skewed"), (4096, 1, 64, "skewed"),
    (700, 64, 100, "flat"), (2049, 2, 1023, "skewed"), (9001, 8, 33, "far"), (3000, 2, 4, "none"), (500, 2, 9, "same"),
    (16384, 2, 64, "skewed"), (16385, 2, 1000, "far"), (100003, 3, 11, "skewed")])
def test_expert_order(tokens, top, experts, kind):
    from originccl_b200.ops import experts as ex
    for itype in (torch.int32, torch.int64):
        ids = torch.full((tokens, top), -1, device="cuda", dtype=itype) if kind == "none" else \
            some_ids(tokens * top, experts, kind, 3, itype).reshape(tokens, top)
        order = ex.sort_by_expert(ids, experts)
        slots, sources, offsets, kept = order64(ids, experts)
        assert order.slots.reshape(-1).tolist() == slots and order.sources.tolist() == sources
        if offsets is not None:
            assert order.offsets.tolist() == offsets
        assert order.offsets[-1].item() == kept and order.offsets[0].item() == 0
        assert (order.offsets.diff() >= 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("tokens,top,experts,h,kind", [
    (1, 1, 1, 1, "flat"), (8, 2, 8, 4096, "flat"), (33, 3, 7, 251, "far"), (129, 8, 64, 1000, "skewed"), (40, 9, 12, 2056, "far"),
    (5, 64, 100, 72, "flat"), (17, 2, 4, 64, "none"), (6, 2, 5, 9001, "far"), (700, 1, 3, 40, "same")])
def test_experts(dtype, tokens, top, experts, h, kind):
    from originccl_b200.ops import experts as ex
    ids = torch.full((tokens, top), -1, device="cuda") if kind == "none" else \
        some_ids(tokens * top, experts, kind, 3).reshape(tokens, top)
    order = ex.sort_by_expert(ids, experts)
    slots = order.slots.long()
    kept = (slots >= 0)[..., None]
    at = slots.clamp(min=0)
    nkept = int(order.offsets[-1])
    src = order.sources[:nkept].long()
    x, rows, dy = randn((tokens, h), dtype, 4), randn((tokens * top, h), dtype, 5), randn((tokens, h), dtype, 6)
    got = ex.dispatch_forward(x, order)
    assert torch.equal(got[:nkept], x[src // top]) and got[nkept:].eq(0).all()
    rows[nkept:] = float("nan")  # behind the last row: not read
    picked = torch.where(kept, torch.nan_to_num(rows.double())[at], 0.0)
    for wtype in (dtype, torch.float32, None):
        w = None if wtype is None else randn((tokens, top), wtype, 7)
        if w is not None:
            w[slots < 0] = float("nan")  # weights of dropped assignments: not used
        w64 = torch.where(kept, 1.0 if w is None else w.double()[..., None], 0.0)
        y = ex.combine_forward(rows, order, w)
        terms = picked * w64
        check(y, terms.sum(1), (top + 1) * U * terms.abs().sum(1), "combine")
        drows, dw = ex.combine_backward(dy, rows, order, w)
        exact = (dy.double()[:, None] * w64).reshape(tokens * top, h)
        check(drows[:nkept], exact[src], 2 * U * exact[src].abs(), "drows")
        assert drows[nkept:].eq(0).all()
        if w is None:
            assert dw is None
        else:  # a lane adds h / 128 + 8 products in a register, the trees over registers and lanes 7
            dots = picked * dy.double()[:, None]
            check(dw, dots.sum(-1), (h / 128 + 16) * U * dots.abs().sum(-1), "dweights")
    drows = torch.where(torch.arange(tokens * top, device="cuda")[:, None] < nkept, rows, torch.full_like(rows, float("nan")))
    check(ex.dispatch_backward(drows, order), picked.sum(1), (top + 1) * U * picked.abs().sum(1), "dx")


def test_expert_layouts_and_nothing():
    from originccl_b200.ops import experts as ex
    order = ex.sort_by_expert(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 6)
    assert order.offsets.eq(0).all() and order.slots.shape == (0, 2)
    x = torch.empty(0, 16, device="cuda")
    rows = ex.dispatch_forward(x, order)
    w = torch.empty(0, 2, device="cuda")
    assert rows.shape == (0, 16) and ex.combine_forward(rows, order, w).shape == (0, 16)
    drows, dw = ex.combine_backward(x, rows, order, w)
    assert drows.shape == (0, 16) and dw.shape == (0, 2)
    ids = some_ids(60, 6, "flat", 1).reshape(2, 30).t()  # not contiguous
    order = ex.sort_by_expert(ids, 6)
    same = ex.sort_by_expert(ids.contiguous(), 6)
    assert order.num_experts == 6
    for name in ("slots", "sources", "offsets"):
        assert torch.equal(getattr(order, name), getattr(same, name))
    assert order.rank_counts(3).sum().item() == 60 and order.rank_counts(3).shape == (3,)
    wide = randn((30, 70), torch.bfloat16, 2)
    for view in (wide[:, 3:43], wide[:, 8:48], wide[:1, :40].expand(30, 40), wide.t()[:40].t()):
        assert torch.equal(ex.dispatch_forward(view, order), ex.dispatch_forward(view.contiguous(), order))
        rows, w = randn((60, 40), torch.bfloat16, 3), randn((30, 2), torch.float32, 4)
        a, b = ex.combine_backward(view, rows, order, w), ex.combine_backward(view.contiguous(), rows, order, w)
        # aligned and misaligned rows sum dweights in another order
        assert torch.equal(a[0], b[0])
        dots = (rows[order.slots.long()].double() * view.double()[:, None])
        check(a[1], dots.sum(-1), 48 * U * dots.abs().sum(-1))
    buf = torch.zeros(62, 40, device="cuda", dtype=torch.bfloat16)
    ex.dispatch_forward(wide[:, :40], order, out=buf[1:61])
    assert torch.equal(buf[1:61], ex.dispatch_forward(wide[:, :40], order)) and buf[0].eq(0).all() and buf[61].eq(0).all()


def test_expert_gradients_against_differences():
    """Dispatch and combine are linear in their rows and in the weights."""
    from originccl_b200.ops import experts as ex
    ids = some_ids(80, 5, "far", 1).reshape(40, 2)
    order = ex.sort_by_expert(ids, 5)
    x, w, t = randn((40, 96), torch.float32, 2), randn((40, 2), torch.float32, 3), randn((40, 96), torch.float32, 4)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    (ex.combine(ex.dispatch(xs, order) * 2.0, order, ws) * t).sum().backward()
    keep = (order.slots >= 0).double()
    f = lambda x, w: ((x * 2.0)[:, None] * (w * keep)[..., None] * t.double()[:, None]).sum()  # noqa: E731
    for grad, v, hi in ((xs.grad, randn((40, 96), torch.float64, 5), lambda v: f(x.double() + v, w.double())),
                        (ws.grad, randn((40, 2), torch.float64, 6), lambda v: f(x.double(), w.double() + v))):
        want = hi(v) - f(x.double(), w.double())
        assert abs((grad.double() * v).sum() - want) <= 64 * U * (grad.double() * v).abs().sum() + 40 * 96 * U


# ---------------------------------------------------------------- gradient norm and clipping
def clip64(grads, max_norm, eps=1e-6):
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    return norm, min(1.0, max_norm / (float(norm) + eps))


def check_clip(grads, max_norm, outs=None):
    """m = 64 + 1: a thread adds 64 squares in 32 bits and the rest in 64; the norm has half that error, and
    the coefficient and the product round three more times."""
    from originccl_b200.ops import gradients
    before = [g.clone() for g in grads]
    norm64, coef = clip64(grads, max_norm)
    norm = gradients.clip_grad_norm(grads, max_norm, outs=outs)
    check(norm, norm64, 34 * U * norm64, "norm")
    for g, b, o in zip(grads, before, grads if outs is None else outs):
        exact = b.double() * coef
        check(o, exact, 40 * U * exact.abs())
        if outs is not None:
            assert torch.equal(g, b)
    return coef


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [2048], [4099, 1, 17], [70000, 33, 1], [1 << 20], [7] * 40, [1000] * 300,
                                   [5] * 2500])
def test_clip(dtype, sizes):
    for off in (0, 3):  # tensors at any alignment in one flat storage
        flat = randn(sum(sizes) + off, dtype, 1)
        grads = list(torch.split(flat[off:], sizes))
        bound = 0.4 * float(flat[off:].double().norm())
        assert check_clip([g.clone() for g in grads], bound) < 1.0
        guard = flat[:off].clone()
        check_clip(grads, bound)  # in place
        assert torch.equal(flat[:off], guard)
        flat = randn(sum(sizes) + off, dtype, 2)
        grads = list(torch.split(flat[off:], sizes))
        for otype in {dtype, torch.float32}:
            for shift in (0, 1):
                store = torch.full((sum(sizes) + shift + 1,), 9.0, device="cuda", dtype=otype)
                outs = list(torch.split(store[shift:-1], sizes))
                check_clip(grads, 0.4 * math.sqrt(sum(sizes)), outs)
                assert store[:shift].eq(9).all() and store[-1:].eq(9).all()
                assert check_clip(grads, 9.0 * math.sqrt(sum(sizes)) + 9, outs) == 1.0
                assert all(torch.equal(o, g.to(otype)) for o, g in zip(outs, grads))


def test_clip_mixed_types_layouts_and_the_norm_alone():
    from originccl_b200.ops import gradients
    grads = [randn((30, 50), torch.bfloat16, 1), randn(17, torch.float32, 2), randn((4, 5, 6), torch.float16, 3),
             randn((50, 30), torch.float32, 4).t(), randn((2, 3, 4, 5), torch.bfloat16, 5).permute(0, 2, 3, 1)]
    norm64, _ = clip64(grads, 1.0)
    check(gradients.grad_norm(grads), norm64, 34 * U * norm64)
    check_clip(grads, 3.0, [torch.empty_like(g, dtype=torch.float32) for g in grads])
    check_clip(grads, 3.0)
    same = randn((64, 64), torch.bfloat16, 6)
    check(gradients.grad_norm([same, same]), (2 * same.double().square().sum()).sqrt(), 34 * U * 2 ** 0.5 * same.double().norm())
    assert gradients.grad_norm([torch.empty(0, device="cuda")]).item() == 0.0


def test_clip_of_values_that_are_not_finite():
    """As torch.nn.utils.clip_grad_norm_: an infinite norm makes the factor 0, a NaN one NaN."""
    from originccl_b200.ops import gradients
    for bad in (float("inf"), float("nan")):
        g = randn(5000, torch.float32, 1)
        g[77] = bad
        want = g.clone().requires_grad_()
        want.grad = g.clone()
        n = torch.nn.utils.clip_grad_norm_([want], 1.0)
        m = gradients.clip_grad_norm([g], 1.0)
        assert torch.equal(m.isnan(), n.isnan()) and torch.equal(m.isinf(), n.isinf())
        assert torch.equal(g.isnan(), want.grad.isnan()) and g[~g.isnan()].eq(0).all()
    g = torch.zeros(100, device="cuda")
    assert gradients.clip_grad_norm([g], 0.0).item() == 0.0 and g.eq(0).all()
    g = torch.ones(100, device="cuda")
    gradients.clip_grad_norm([g], 0.0)
    assert g.eq(0).all()


def test_norm_is_the_same_on_every_run_and_over_two_types_of_list():
    from originccl_b200.ops import gradients
    flat = randn(3_000_001, torch.bfloat16, 1)
    first = gradients.grad_norm([flat])
    assert all(torch.equal(gradients.grad_norm([flat]), first) for _ in range(5))


def test_sharded_norm_uses_the_communicator():
    import originccl_b200 as occl
    from originccl_b200.ops import gradients
    comm = occl.Communicator().init(0, 1, None, device=0)
    g = randn(1000, torch.float32, 1)
    assert torch.equal(gradients.grad_norm([g], comm=comm), gradients.grad_norm([g]))

    class Twice:  # stands for two ranks that hold equal shards
        world_size = 2

        def all_reduce(self, t):
            comm.all_reduce(t, scale=2.0)

    norm = gradients.clip_grad_norm([g.clone()], 1.0, comm=Twice())
    check(norm, g.double().norm() * 2 ** 0.5, 34 * U * g.double().norm() * 2 ** 0.5)
    comm.destroy()


# ---------------------------------------------------------------- streams, graphs
def all_ops(seed):
    """One call of everything on inputs of a seed: (function, list of its inputs)."""
    from originccl_b200.ops import embedding, experts as ex, gradients, norm
    x, w, b = randn((200, 520), torch.bfloat16, seed), randn(520, torch.bfloat16, seed + 1), randn(520, torch.bfloat16, seed + 2)
    dy = randn((200, 520), torch.bfloat16, seed + 3)
    ids = some_ids(200, 1500, "skewed", seed + 4)
    who = some_ids(400, 9, "far", seed + 5).reshape(200, 2)
    cw = randn((200, 2), torch.float32, seed + 6)
    ins = [x, w, b, dy, ids, who, cw]

    def call():
        y, mean, rstd = norm.layer_norm_forward(x, w, b)
        out = [y, mean, rstd, *norm.layer_norm_backward(dy, x, mean, rstd, w)]
        z, r = norm.rms_norm_forward(x, w)
        out += [z, r, *norm.rms_norm_backward(dy, x, r, w)]
        out += [embedding.embedding_forward(ids, x, 0.5), embedding.embedding_backward(dy, ids, 1500, 0.5)]
        order = ex.sort_by_expert(who, 9)
        rows = ex.dispatch_forward(x, order)
        out += [order.slots, order.sources, order.offsets, rows, ex.combine_forward(rows, order, cw), *ex.combine_backward(dy, rows, order, cw),
                ex.dispatch_backward(rows, order)]
        outs = [torch.empty_like(t) for t in (x, dy)]
        out += [gradients.clip_grad_norm([x, dy], 1.0, outs=outs), *outs]
        return out
    return call, ins


def equal(a, b):
    return len(a) == len(b) and all(torch.equal(p.reshape(-1).view(torch.uint8), q.reshape(-1).view(torch.uint8))
                                    for p, q in zip(a, b))


def test_two_captured_graphs_replay_on_two_streams():
    from originccl_b200.utils.graphs import capture
    graphs = []
    for seed in (10, 50):
        call, ins = all_ops(seed)
        box = {}

        def fn(call=call, box=box):
            box["out"] = call()
        graphs.append((capture(fn), ins, box))
    for seed in (100, 200):  # new inputs in the captured buffers
        for i, (_, ins, _) in enumerate(graphs):
            for t, new in zip(ins, all_ops(seed + 40 * i)[1]):
                t.copy_(new)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(3):
            for s, (g, _, _) in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for i, (_, _, box) in enumerate(graphs):
            want = all_ops(seed + 40 * i)[0]()
            assert equal(box["out"], want)


def test_calls_on_other_streams_run_there():
    call, _ = all_ops(300)
    want = call()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        a = call()
    with torch.cuda.stream(t):
        b = call()
    torch.cuda.synchronize()
    assert equal(a, want) and equal(b, want)


# ---------------------------------------------------------------- together
def test_a_training_step_on_the_operators():
    """The small stack with a table, its gradients in buckets, synced and clipped; against the same
    stack on torch's operators. Every stage is off by a few roundings of its sums' magnitudes (hidden
    and ffn below 1024 terms): 2^-24 x 4096 of the largest gradient bounds the whole chain."""
    import originccl_b200 as occl
    from originccl_b200.models import TinyLlamaStack
    from originccl_b200.parallel import DataParallelSync, GradBuckets
    ids = some_ids(600, 1024, "skewed", 1).reshape(4, 150)
    comm = occl.Communicator().init(0, 1, None, device=0)
    results = []
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        for native in (False, True):
            m = TinyLlamaStack(hidden=256, ffn=768, layers=2, device="cuda", seed=5, vocab=1024, native=native)
            buckets = GradBuckets(m.named_parameters(), bucket_bytes=1 << 18)
            dp = DataParallelSync(comm, buckets)
            m(ids).square().mean().backward()
            dp.sync()
            plain = [p.grad.clone() for p in m.parameters()]
            norm = dp.clip_grad_norm_(0.01)
            n64, coef = clip64(plain, 0.01)
            check(norm, n64, 34 * U * n64)
            assert coef < 1.0
            for p, g in zip(m.parameters(), plain):
                check(p.grad, g.double() * coef, 40 * U * g.double().abs())
            results.append((dict(m.named_parameters()), plain))
            dp.close()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = old
    comm.destroy()
    (names, torch_grads), (_, grads) = results
    for name, a, b in zip(names, torch_grads, grads):
        assert (a - b).abs().max() <= 4096 * U * a.abs().max(), name


def test_tokens_go_to_their_experts_and_back():
    """Sort, dispatch, the exchange (one rank), a GEMM per expert, combine; and the gradients."""
    import originccl_b200 as occl
    from originccl_b200.ops import experts as ex, gemm
    if not gemm.available():
        pytest.skip("needs an sm_100 GPU")
    comm = occl.Communicator().init(0, 1, None, device=0)
    tokens, top, n, h = 150, 2, 4, 128
    ids = some_ids(tokens * top, n, "far", 3).reshape(tokens, top)
    x, w = randn((tokens, h), torch.bfloat16, 4), randn((tokens, top), torch.float32, 5)
    mats = randn((n, h, h), torch.bfloat16, 6, 0.1)
    order = ex.sort_by_expert(ids, n)
    send = ex.dispatch(x, order)
    recv = torch.empty_like(send)
    comm.all_to_all(recv, send)
    answers = torch.zeros_like(recv)
    ends = order.offsets.tolist()
    for e in range(n):
        if ends[e + 1] > ends[e]:
            answers[ends[e]:ends[e + 1]] = gemm.gemm(recv[ends[e]:ends[e + 1]], mats[e])
    assert gemm.check_error() == 0
    y = ex.combine(answers, order, w)
    kept = (ids >= 0) & (ids < n)
    exact = torch.zeros(tokens, h, dtype=torch.float64, device="cuda")
    size = exact.clone()
    for j in range(top):
        m = mats.double()[ids[:, j].clamp(0, n - 1)]
        term = torch.einsum("th,tkh->tk", x.double(), m) * (w.double() * kept)[:, j, None]
        bound = torch.einsum("th,tkh->tk", x.double().abs(), m.abs()) * (w.double().abs() * kept)[:, j, None]
        exact += term
        size += 2.0 ** -8 * term.abs() + (h + 8) * U * bound  # an answer is rounded to bf16 once
    check(y, exact, size)
    comm.destroy()


# ---------------------------------------------------------------- refusals that need a GPU, large offsets
def test_overlapping_tensors_are_not_clipped():
    from originccl_b200.ops import gradients
    flat = randn(1000, torch.float32, 1)
    keep = flat.clone()
    for grads, outs in (([flat[:600], flat[500:]], None),               # overlap in place
                        ([flat, flat], None),                           # the same tensor twice
                        ([flat[:400], flat[400:800]], [flat[100:500], flat[600:]]),
                        ([flat[:100], flat[100:200]], [flat[100:200], flat[:100]]),  # each other's place
                        ([flat[:100], flat[100:200]], [torch.empty(100, device="cuda")] * 2)):
        if outs is not None and [o.numel() for o in outs] != [g.numel() for g in grads]:
            outs = [o[:g.numel()] for o, g in zip(outs, grads)]
        with pytest.raises(ValueError, match="overlap"):
            gradients.clip_grad_norm(grads, 1e-3, outs=outs)
    with pytest.raises(TypeError, match="float32"):
        gradients.clip_grad_norm([flat], 1.0, outs=[torch.empty(1000, device="cuda", dtype=torch.float16)])
    with pytest.raises(ValueError, match="shape"):
        gradients.clip_grad_norm([flat], 1.0, outs=[torch.empty(10, 100, device="cuda")])
    with pytest.raises(ValueError, match="dense"):
        gradients.clip_grad_norm([flat[::2]], 1.0)
    with pytest.raises(ValueError, match="one device"):
        gradients.clip_grad_norm([flat, torch.zeros(3)], 1.0)
    assert torch.equal(flat, keep)
    gradients.clip_grad_norm([flat[:0], flat[:0], flat], 1e-3, outs=None)  # empty tensors share nothing
    assert not torch.equal(flat, keep)


def test_outputs_that_are_written_count_as_changed():
    """Autograd notices that a tensor it saved was written by an operator."""
    from originccl_b200.ops import gradients, norm
    x = randn((4, 64), torch.float32, 1)
    a = torch.ones(4, 64, device="cuda", requires_grad=True)
    y = a * x
    norm.rms_norm_forward(x, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    before = x._version
    gradients.clip_grad_norm([x], 1.0)
    assert x._version > before


def test_offsets_beyond_32_bits():
    from originccl_b200.ops import embedding, experts as ex, gradients, norm
    rows, h = 600_000, 4096  # 2.46e9 elements
    big = torch.zeros(rows, h, device="cuda", dtype=torch.bfloat16)
    ids = torch.tensor([0, rows - 1, rows - 1, rows - 7], device="cuda")
    big[-8:] = randn((8, h), torch.bfloat16, 1)
    assert torch.equal(embedding.embedding_forward(ids, big), big[ids])
    y, rstd = norm.rms_norm_forward(big)
    check(y[-8:], norm64("rms", big[-8:], None, None, 1e-5)[0], 64 * U * big[-8:].double().abs().amax() * 2)
    assert y[:-8].abs().amax() == 0
    dx, _ = norm.rms_norm_backward(big, big, rstd)
    assert dx[:-8].abs().amax() == 0 and dx[-8:].abs().amax() > 0
    total = gradients.clip_grad_norm([big], 1.0, outs=[y])
    exact = big[-8:].double().norm()
    check(total, exact, 34 * U * exact)
    check(y[-8:], big[-8:].double() / (float(exact) + 1e-6), 40 * U * big[-8:].double().abs())
    del y, dx
    dy = randn((4, h), torch.bfloat16, 2)
    grad = embedding.embedding_backward(dy, ids, rows, out=big)
    assert torch.equal(grad[0], dy[0]) and torch.equal(grad[rows - 7], dy[3]) and grad[1:rows - 7].abs().amax() == 0
    check(grad[rows - 1], dy[1].double() + dy[2].double(), 2 * U * (dy[1].double().abs() + dy[2].double().abs()))
    order = ex.sort_by_expert(torch.arange(rows, device="cuda").remainder(2).reshape(-1, 2), 2)
    x = torch.arange(rows // 2, device="cuda", dtype=torch.float32)[:, None].remainder(251).to(torch.bfloat16).expand(-1, h)
    ex.dispatch_forward(x, order, out=big)
    assert torch.equal(big[:, 0], x[order.sources.long() // 2, 0]) and torch.equal(big[:, 0], big[:, -1])
    assert torch.equal(ex.combine_forward(big, order), x.contiguous() * 2)


def test_a_backward_pass_is_captured():
    from originccl_b200.ops import norm
    from originccl_b200.utils.graphs import capture
    x = randn((64, 256), torch.float32, 1).requires_grad_()
    w = randn(256, torch.float32, 2).requires_grad_()
    t = randn((64, 256), torch.float32, 3)
    x.grad, w.grad = torch.zeros_like(x), torch.zeros_like(w)

    def step():
        x.grad.zero_()
        w.grad.zero_()
        (norm.rms_norm(x, w) * t).sum().backward()
    step()
    g = capture(step)
    want = []
    for seed in (4, 5):
        with torch.no_grad():
            x.copy_(randn((64, 256), torch.float32, seed))
        g.replay()
        torch.cuda.synchronize()
        got = x.grad.clone(), w.grad.clone()
        _, rstd = norm.rms_norm_forward(x.detach(), w.detach())
        want = norm.rms_norm_backward(t, x.detach(), rstd, w.detach())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_outputs_in_their_inputs_are_refused():
    from originccl_b200.ops import embedding, experts as ex, norm
    buf = randn(4096, torch.float32, 1)
    x = buf[:1024].view(16, 64)
    with pytest.raises(ValueError, match="overlap"):
        norm.rms_norm_forward(x, out=buf[64:1088].view(16, 64))
    with pytest.raises(ValueError, match="overlap"):
        norm.rms_norm_forward(x, buf[1000:1064], out=buf[1024:2048].view(16, 64))
    ids = torch.zeros(16, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        embedding.embedding_forward(ids, x, out=x)
    with pytest.raises(ValueError, match="overlap"):
        embedding.embedding_backward(x, ids, 16, out=x)
    order = ex.sort_by_expert(ids, 2)
    with pytest.raises(ValueError, match="overlap"):
        ex.dispatch_forward(x, order, out=buf[960:1984].view(16, 64))
    ex.dispatch_forward(x, order, out=buf[1024:2048].view(16, 64))


# ---------------------------------------------------------------- the C interface where Python takes a narrower road
@pytest.mark.parametrize("dtype,wtype,rows,h", [
    (torch.bfloat16, torch.float32, 3, 64), (torch.bfloat16, torch.bfloat16, 700, 4096), (torch.float16, torch.float32, 700, 4096),
    (torch.float16, torch.float32, 3000, 1001), (torch.bfloat16, torch.float32, 400, 9000), (torch.float32, torch.float32, 700, 4096),
    (torch.float32, torch.float32, 2, 40000)])
def test_layer_norm_with_a_bias_and_no_weight(dtype, wtype, rows, h):
    """Each of weight and bias may be missing, in every form of the kernel. m as in check_norm."""
    from originccl_b200 import _native
    code = {torch.float32: 0, torch.bfloat16: 4, torch.float16: 5}
    x, b = randn((rows, h), dtype, 1, 2.0, 0.5), randn(h, wtype, 2, 0.3)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    rc = _native.lib().bcclNormForward(0, x.data_ptr(), h, None, b.data_ptr(), y.data_ptr(), h, mean.data_ptr(), rstd.data_ptr(),
                                       rows, h, 1e-5, code[dtype], code[wtype], torch.cuda.current_stream().cuda_stream)
    assert rc == 0, _native.last_error()
    y64, mean64, rstd64, xh = norm64("layer", x, None, b, 1e-5)
    size = x.double().abs().mean(-1, keepdim=True) * rstd64[:, None]
    m = 64 * U
    check(y, y64, m * (xh.abs() + size) + 2 * U * b.double().abs(), "y")
    check(mean, mean64, m * x.double().abs().mean(-1), "mean")
    check(rstd, rstd64, m * rstd64 * (1 + size[:, 0] ** 2 * U), "rstd")


def ring_pair():
    """Rows of two widths that one instance of the ring kernels takes, with different amounts of shared memory."""
    return [(randn((rows, h), torch.bfloat16, h), randn(h, torch.bfloat16, h + 1), randn((rows, h), torch.bfloat16, h + 2))
            for rows, h in ((400, 8192), (1500, 2048))]


def both_ways(x, w, dy):
    from originccl_b200.ops import norm
    y, rstd = norm.rms_norm_forward(x, w)
    return [y, rstd, *norm.rms_norm_backward(dy, x, rstd, w)]


def test_norms_of_two_widths_in_two_threads():
    """Calls on different streams may run at the same time: a narrow one takes nothing from a wide one
    between its setup and its launch."""
    import threading
    data = ring_pair()
    want = [both_ways(*d) for d in data]
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(4)

    def work(i):
        try:
            start.wait(60)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(400):
                    got = both_ways(*data[i])
                torch.cuda.current_stream().synchronize()
            assert equal(got, want[i])
        except BaseException as e:  # reported by the main thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i % 2,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not failed and not any(t.is_alive() for t in threads), failed


def test_norms_of_two_widths_in_one_graph():
    from originccl_b200.utils.graphs import capture
    data, box = ring_pair(), {}

    def fn():
        box["out"] = [t for d in data for t in both_ways(*d)]
    g = capture(fn)
    both_ways(*(t[:, :1024].contiguous() if t.dim() == 2 else t[:1024] for t in data[1]))  # narrower still, before the replay
    g.replay()
    torch.cuda.synchronize()
    assert equal(box["out"], [t for d in data for t in both_ways(*d)])


def test_norm_launches_of_two_widths_in_threads_never_fail():
    """The same through the C interface, whose calls run without the interpreter's lock, often enough for
    the threads to meet: about 1 wide call in 400 failed where each call set a limit of its own."""
    import sys
    import threading
    from originccl_b200 import _native
    forward = _native.lib().bcclNormForward
    failed = [0] * 4

    def work(i, x, w):
        (rows, h), s = x.shape, torch.cuda.Stream()
        y, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
        args = (1, x.data_ptr(), h, w.data_ptr(), None, y.data_ptr(), h, None, rstd.data_ptr(), rows, h, 1e-5, 4, 4, s.cuda_stream)
        for k in range(10000):
            failed[i] += forward(*args) != 0
            if k % 200 == 199:
                s.synchronize()
    data = ring_pair()
    torch.cuda.synchronize()
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=(i, *data[i % 2][:2])) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(120)
    finally:
        sys.setswitchinterval(interval)
    torch.cuda.synchronize()
    assert not any(t.is_alive() for t in threads) and failed == [0] * 4


def test_a_model_serves_without_a_graph():
    """The stack in inference mode and under no_grad, eager and captured, also while a training step's loss
    is still held: the same bits as its recorded forward pass."""
    from originccl_b200.models import TinyLlamaStack
    from originccl_b200.ops import experts as ex, norm
    from originccl_b200.utils.graphs import capture
    m = TinyLlamaStack(hidden=256, ffn=768, layers=2, device="cuda", dtype=torch.bfloat16, seed=5, vocab=1024, native=True)
    ids = some_ids(64, 1024, "skewed", 1)
    want = m(ids)
    loss = want.square().mean()  # held until the end
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            assert torch.equal(m(ids), want)
    w = torch.ones(256, device="cuda", requires_grad=True)
    b = torch.zeros(256, device="cuda", requires_grad=True)
    order = ex.sort_by_expert(ids[:, None].remainder(4), 4)
    share = torch.full((64, 1), 0.5, device="cuda", requires_grad=True)
    held = norm.layer_norm(want, w, b), ex.combine(ex.dispatch(want, order), order, share)
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            assert torch.equal(norm.layer_norm(want, w, b), held[0])
            assert torch.equal(ex.combine(ex.dispatch(want, order), order, share), held[1])
    box = {}

    @torch.no_grad()
    def serve():
        box["y"] = m(ids), norm.layer_norm(want, w, b)
    g = capture(serve)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(box["y"][0], want) and torch.equal(box["y"][1], held[0])
    loss.backward()
    assert m.embed.grad.abs().amax() > 0


def test_a_capture_beside_another_operators_graph_is_refused():
    """torch's own operator made the weight's accumulation node on the default stream, and its result is
    held: the captured forward pass is refused, before a backward pass could be captured."""
    from originccl_b200.ops import norm
    from originccl_b200.utils.graphs import capture
    x, w = randn((64, 256), torch.float32, 1), randn(256, torch.float32, 2).requires_grad_()
    held = (w * 2).sum()
    with pytest.raises(RuntimeError, match="still alive"):
        capture(lambda: norm.rms_norm(x, w), warmup=0)
    del held
    box = {}

    def fn():
        box["y"] = norm.rms_norm(x, w)
    g = capture(fn, warmup=0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(box["y"].detach(), norm.rms_norm_forward(x, w.detach())[0])
    del box["y"]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        held = (w * 3).sum()
    norm.rms_norm(x, w)  # marks that node, from the default stream: still the node's stream
    with pytest.raises(RuntimeError, match="still alive"):
        capture(lambda: norm.rms_norm(x, w), warmup=0)
    del held


@pytest.mark.parametrize("clip", [False, True])
def test_replicated_gradients_count_once(clip):
    """Mixed types, some of them held by both of two ranks (stood in for by a doubled sum)."""
    import originccl_b200 as occl
    from originccl_b200.ops import gradients
    comm = occl.Communicator().init(0, 1, None, device=0)

    class Twice:
        world_size = 2

        def all_reduce(self, t):
            comm.all_reduce(t, scale=2.0)

    grads = [randn(1000, torch.float32, 1), randn((30, 41), torch.bfloat16, 2), randn(7, torch.float32, 3), randn(5000, torch.bfloat16, 4),
             torch.empty(0, device="cuda"), randn(33, torch.float16, 5)]
    for flags in ([False, True, True, False, True, False], [True] * 6, [False] * 6, [0, 0, 0, 0, 1, 0]):
        mine = [g.clone() for g in grads]
        n64 = sum(g.double().square().sum() * (1 if r else 2) for g, r in zip(grads, flags)).sqrt()
        if clip:
            norm = gradients.clip_grad_norm(mine, 3.0, comm=Twice(), replicated=flags)
            for m, g in zip(mine, grads):
                exact = g.double() * (3.0 / (float(n64) + 1e-6))
                check(m, exact, 40 * U * exact.abs())
        else:
            norm = gradients.grad_norm(mine, comm=Twice(), replicated=flags)
        check(norm, n64, 34 * U * n64)
    comm.destroy()


@pytest.mark.parametrize("h", [2 ** 23, 2 ** 23 - 1])
def test_embedding_of_the_longest_rows(h):
    """A token over several windows, so that its partial rows are joined."""
    from originccl_b200.ops import embedding
    ids = torch.tensor([1] * 15 + [0, 1], device="cuda")
    w = randn((2, h), torch.float32, 1)
    assert torch.equal(embedding.embedding_forward(ids[-2:], w), w[ids[-2:]])
    dy = randn((17, h), torch.float32, 2)
    got = embedding.embedding_backward(dy, ids, 3)
    for row in range(3):
        terms = dy[ids == row].double()
        check(got[row], terms.sum(0), (terms.shape[0] + 2) * U * terms.abs().sum(0))


@pytest.mark.parametrize("rows,h,gap", [(40, 640, 0), (40, 651, 1), (3000, 1016, 8), (3000, 1001, 3)])
def test_outputs_beside_their_inputs_in_one_array(rows, h, gap):
    """Columns of one array, either of them first, at any alignment; but not a column of the input's. The same
    bits as from and into arrays of their own with that alignment (which decides which thread adds what)."""
    from originccl_b200.ops import embedding, norm
    wide = randn((rows, 2 * h + 2 * gap), torch.bfloat16, 1)
    w = randn(h, torch.bfloat16, 2)
    ids = some_ids(rows, rows, "flat", 3)
    for a, b in ((gap, h + gap), (h + gap, gap)):
        for call in (lambda x, out: norm.rms_norm_forward(x, w, out=out)[0], lambda x, out: norm.layer_norm_forward(x, w, out=out)[0],
                     lambda x, out: embedding.embedding_forward(ids, x, 0.5, out=out)):
            buf = wide.clone()
            x, out = buf[:, a:a + h], buf[:, b:b + h]
            want = call(wide[:, a:a + h], torch.empty_like(wide)[:, b:b + h])
            assert call(x, out) is not None and torch.equal(out, want)
            out.copy_(wide[:, b:b + h])
            assert torch.equal(buf, wide)  # nothing else was written
            for off in (-1, 1):
                if (off < 0) == (a < b):  # one column into the input
                    with pytest.raises(ValueError, match="overlap"):
                        call(x, buf[:, b + off:b + off + h])


# Rows per block of the ring kernels: more than the ring is deep, at both accesses per thread, at rows that begin
# on 16 bytes and at rows that do not.
RINGS = [(torch.bfloat16, 9000, 1531), (torch.float16, 9000, 1528), (torch.float16, 3000, 4097), (torch.bfloat16, 1000, 8200),
         (torch.float16, 1000, 8201), (torch.bfloat16, 1000, 16384), (torch.bfloat16, 1000, 16001), (torch.float32, 3000, 2049),
         (torch.float32, 2500, 4096), (torch.float32, 1000, 8189), (torch.bfloat16, 20000, 140), (torch.float32, 20000, 71)]


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype,rows,h", RINGS)
def test_norms_of_many_rows(kind, dtype, rows, h):
    x, dy = randn((rows, h), dtype, 3, 2.0, 0.5), randn((rows, h), dtype, 4, 0.1)
    for wtype in {dtype, torch.float32}:
        w, b = randn(h, wtype, 1, 0.2, 1.0), randn(h, wtype, 2, 0.3)
        check_norm(kind, x, w, b if kind == "layer" else None, 1e-5, dy)
    check_norm(kind, x, None, None, 1e-5, dy)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype,rows,h", RINGS[:6])
def test_norms_of_many_rows_in_other_layouts(kind, dtype, rows, h):
    """Rows of x, dy or both that begin elsewhere than those of y and dx; and all at the same odd distance."""
    wide, other = randn((rows, h + 19), dtype, 3, 2.0, 0.5), randn((rows, h + 19), dtype, 4, 0.1)
    w = randn(h, dtype, 1, 0.2, 1.0)
    for x, dy in ((wide[:, 5:h + 5], other[:, :h]), (wide[:, :h].contiguous(), other[:, 1:h + 1]),
                  (wide[:, 8:h + 8], other[:, 8:h + 8].contiguous()), (wide[:, :h].contiguous(), other[:1, :h].expand(rows, h))):
        check_norm(kind, x, w, None, 1e-5, dy)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype,rows,h", RINGS + [(torch.bfloat16, 37, 1531), (torch.float16, 3, 40001), (torch.float32, 500, 33)])
def test_norms_in_place(kind, dtype, rows, h):
    """The same bits as into an array of its own, whatever a block's neighbours write meanwhile."""
    from originccl_b200.ops import norm
    w, b = randn(h, dtype, 1, 0.2, 1.0), randn(h, dtype, 2, 0.3)
    run = (lambda x, out: norm.layer_norm_forward(x, w, b, out=out)) if kind == "layer" else \
        (lambda x, out: norm.rms_norm_forward(x, w, out=out))
    for off in (0, 3):  # rows that begin anywhere
        store = randn(rows * h + off, dtype, 3, 2.0, 0.5)
        x = store[off:].view(rows, h)
        want = run(x, torch.empty_like(store)[off:].view(rows, h))
        for _ in range(3):
            again = store.clone()
            got = run(again[off:].view(rows, h), again[off:].view(rows, h))
            assert equal(got, want) and torch.equal(again[:off], store[:off])


def test_a_capture_beside_an_eager_graph_of_the_operator_is_refused():
    """The operator's own eager pass on the default stream, whose output is held, and then released."""
    from originccl_b200.models import TinyLlamaStack
    from originccl_b200.ops import embedding, experts as ex, norm
    from originccl_b200.utils.graphs import capture
    x = randn((64, 256), torch.float32, 1).requires_grad_()
    w, b = (randn(256, torch.float32, s).requires_grad_() for s in (2, 3))
    ids = some_ids(64, 64, "flat", 4)
    order = ex.sort_by_expert(ids[:, None], 64)
    for call in (lambda: norm.rms_norm(x, w), lambda: norm.layer_norm(x, w, b), lambda: embedding.embedding(ids, x),
                 lambda: ex.dispatch(x, order), lambda: ex.combine(x, order)):
        held = call()
        with pytest.raises(RuntimeError, match="still alive"):
            capture(call, warmup=0)
        del held
        capture(call, warmup=0).replay()
    torch.cuda.synchronize()
    m = TinyLlamaStack(hidden=64, ffn=128, layers=1, device="cuda", seed=5, vocab=64, native=True)
    loss = m(ids).square().mean()
    with pytest.raises(RuntimeError, match="still alive"):
        capture(lambda: m(ids), warmup=0)
    loss.backward()


@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_a_native_stack_answers_as_torchs(dtype):
    """Small activations, where the epsilon decides: torch takes that of its 32-bit arithmetic for every type.
    Each side rounds twice at most (torch before the weights, which are ones): a step apart, and m as in check_norm twice."""
    from originccl_b200.models import TinyLlamaStack
    m = TinyLlamaStack(hidden=256, ffn=256, layers=1, device="cuda", dtype=dtype, native=True)
    x = randn((40, 256), dtype, 1, 0.01)
    n = m.blocks[0]["norm"]
    for eps in (None, 1e-4):
        n.eps = eps
        got, want = m._norm(n, x).double(), n(x).double()
        assert ((got - want).abs() <= (torch.finfo(dtype).eps + 128 * U) * want.abs() + 2 * TINY[dtype]).all()


def test_an_allocation_that_fails_is_torchs_error():
    """What a program that looks for its largest batch catches. torch's allocator refuses by itself (the process'
    share of the memory is set to less than the output), so the device is asked for nothing."""
    from originccl_b200.ops import experts as ex, norm
    row = torch.zeros(1, 1 << 20, device="cuda")
    order = ex.sort_by_expert(torch.zeros(1 << 12, 1, dtype=torch.int32, device="cuda"), 1)
    torch.cuda.synchronize()
    torch.cuda.set_per_process_memory_fraction(0.02)
    try:
        for call in (lambda: norm.rms_norm_forward(row.expand(1 << 12, -1)),  # 16 GB
                     lambda: ex.dispatch_forward(row.expand(1 << 12, -1), order)):
            with pytest.raises(torch.OutOfMemoryError):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    y, _ = norm.rms_norm_forward(row.expand(2, -1))
    torch.cuda.synchronize()
    assert not y.any()
