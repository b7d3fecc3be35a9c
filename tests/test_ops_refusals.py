"""Argument checks of the compute operators and their host path (CPU): wrong types, shapes, devices and
sizes are refused in Python or by the C interface before any pointer reaches a kernel."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from originccl_b200 import _native  # noqa: E402
from originccl_b200.ops import embedding, experts, gradients, norm  # noqa: E402

bf = torch.bfloat16


def test_norms_refuse():
    x, w = torch.zeros(4, 8, dtype=bf), torch.zeros(8, dtype=bf)
    with pytest.raises(TypeError, match="float32"):
        norm.rms_norm_forward(x.double())
    with pytest.raises(TypeError, match="weight"):
        norm.rms_norm_forward(x, w.half())
    with pytest.raises(TypeError, match="bias"):
        norm.layer_norm_forward(x, w, w.float())
    with pytest.raises(TypeError, match="bias"):
        norm.layer_norm_forward(x, None, w)
    with pytest.raises(ValueError, match="shape"):
        norm.layer_norm_forward(x, torch.zeros(7, dtype=bf))
    with pytest.raises(ValueError, match="last dimension"):
        norm.layer_norm_forward(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="last dimension"):
        norm.rms_norm_forward(torch.zeros(()))
    with pytest.raises(ValueError, match="eps"):
        norm.layer_norm_forward(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        norm.layer_norm_forward(x, w, eps=float("nan"))
    with pytest.raises(ValueError, match="CUDA"):
        norm.layer_norm_forward(x, w)
    with pytest.raises(ValueError, match="dy"):
        norm.rms_norm_backward(x.float(), x, torch.zeros(4), w)
    with pytest.raises(ValueError, match="dy"):
        norm.rms_norm_backward(x[:3], x, torch.zeros(4), w)
    with pytest.raises(ValueError, match="rstd"):
        norm.rms_norm_backward(x, x, torch.zeros(3), w)
    with pytest.raises(ValueError, match="mean"):
        norm.layer_norm_backward(x, x, torch.zeros(4, dtype=bf), torch.zeros(4), w)


def test_negated_views_are_refused():
    x = torch._neg_view(torch.zeros(4, 8))
    for call in (lambda: norm.rms_norm_forward(x), lambda: embedding.embedding_forward(torch.zeros(2, dtype=torch.long), x),
                 lambda: experts.dispatch_forward(x, experts.ExpertOrder(
                     *(torch.zeros(n, dtype=torch.int32) for n in ((4, 1), (4,), (3,)))))):
        with pytest.raises(TypeError, match="negated"):
            call()


def test_embedding_refuses():
    ids, w = torch.zeros(5, dtype=torch.int64), torch.zeros(6, 8, dtype=bf)
    with pytest.raises(TypeError, match="ids"):
        embedding.embedding_forward(ids.to(torch.int16), w)
    with pytest.raises(TypeError, match="weight"):
        embedding.embedding_forward(ids, w.double())
    with pytest.raises(ValueError, match="2-D"):
        embedding.embedding_forward(ids, w[0])
    with pytest.raises(ValueError, match="first_row"):
        embedding.embedding_forward(ids, w, first_row=-1)
    with pytest.raises(ValueError, match="CUDA"):
        embedding.embedding_forward(ids, w)
    dy = torch.zeros(5, 8, dtype=bf)
    with pytest.raises(ValueError, match="one row per id"):
        embedding.embedding_backward(dy[:4], ids, 6)
    with pytest.raises(ValueError, match="padding_idx"):
        embedding.embedding_backward(dy, ids, 6, padding_idx=-1)
    with pytest.raises(ValueError, match="padding_idx"):
        embedding.embedding(ids, w, padding_idx=-2)
    with pytest.raises(ValueError, match="num_rows"):
        embedding.embedding_backward(dy, ids, -1)
    with pytest.raises(ValueError, match="accumulate"):
        embedding.embedding_backward(dy, ids, 6, accumulate=True)
    with pytest.raises(TypeError, match="tensor"):
        embedding.embedding_forward([1, 2], w)
    with pytest.raises(TypeError):
        embedding.embedding_forward(ids, w, scale="2")


def test_experts_refuse():
    ids = torch.zeros(5, 2, dtype=torch.int32)
    with pytest.raises(TypeError, match="expert_ids"):
        experts.sort_by_expert(ids.float(), 4)
    with pytest.raises(ValueError, match="experts"):
        experts.sort_by_expert(ids, 1024)
    with pytest.raises(ValueError, match="experts"):
        experts.sort_by_expert(ids, 0)
    with pytest.raises(ValueError, match="per token"):
        experts.sort_by_expert(torch.zeros(5, 65, dtype=torch.int32), 100)
    with pytest.raises(ValueError, match="per token"):
        experts.sort_by_expert(torch.zeros(5, 0, dtype=torch.int32), 100)
    with pytest.raises(ValueError, match="tokens, top"):
        experts.sort_by_expert(ids[None], 4)
    with pytest.raises(ValueError, match="CUDA"):
        experts.sort_by_expert(ids, 4)
    for parts in ((ids.long(), ids.reshape(-1), ids[:, 0]), (ids, ids.reshape(-1)[1:], ids[:, 0].contiguous()),
                  (ids, ids.reshape(-1), ids.reshape(-1)[:1])):
        with pytest.raises(ValueError, match="sort_by_expert"):
            experts.ExpertOrder(*parts)
    order = experts.ExpertOrder(ids, ids.reshape(-1), ids.reshape(-1)[:5])
    assert order.num_experts == 4
    with pytest.raises(ValueError, match="split"):
        order.rank_counts(3)
    with pytest.raises(ValueError, match="CUDA"):
        experts.dispatch_forward(torch.zeros(5, 8), order)
    with pytest.raises(ValueError, match=r"\[5, h\]"):
        experts.dispatch_forward(torch.zeros(4, 8), order)
    with pytest.raises(ValueError, match=r"\[10, h\]"):
        experts.combine_forward(torch.zeros(5, 8), order)
    with pytest.raises(ValueError, match="weights"):
        experts.combine_forward(torch.zeros(10, 8), order, torch.zeros(5, 3))
    with pytest.raises(TypeError, match="weights"):
        experts.combine_forward(torch.zeros(10, 8), order, torch.zeros(5, 2).half())
    with pytest.raises(ValueError, match="rows"):
        experts.combine_backward(torch.zeros(5, 8), torch.zeros(10, 9), order)


def test_clipping_refuses():
    g = torch.ones(4)
    with pytest.raises(ValueError, match="no gradients"):
        gradients.grad_norm([])
    with pytest.raises(ValueError, match="max_norm"):
        gradients.clip_grad_norm([g], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        gradients.clip_grad_norm([g], float("nan"))
    with pytest.raises(ValueError, match="eps"):
        gradients.clip_grad_norm([g], 1.0, eps=-1e-6)
    with pytest.raises(ValueError, match="outs"):
        gradients.clip_grad_norm([g], 1.0, outs=[])
    with pytest.raises(ValueError, match="gradients"):
        gradients.clip_grad_norm([g.double()], 1.0)


def test_host_gradients_are_clipped():
    grads = [torch.full((3, 4), 2.0), torch.full((5,), -1.0, dtype=bf)]
    norm64 = (48.0 + 5.0) ** 0.5
    got = gradients.clip_grad_norm(grads, 1.0)
    assert abs(got.item() - norm64) <= norm64 * 2 ** -23
    assert torch.allclose(grads[0], torch.full((3, 4), 2.0 / norm64), rtol=2 ** -21)
    assert torch.allclose(grads[1].float(), torch.full((5,), -1.0 / norm64), rtol=2 ** -8)
    assert gradients.grad_norm(grads).item() <= 1.0 + 2 ** -8


def p(n):
    return ctypes.c_void_p(n)


def test_the_c_interface_refuses():
    """Bad arguments return an error with a message; no GPU is needed to refuse them."""
    lib = _native.lib()

    def refused(rc, what):
        assert rc != 0 and what in _native.last_error(), _native.last_error()
    one = (ctypes.c_size_t * 1)(4)
    tensor = (ctypes.c_void_p * 1)(64)
    odd = (ctypes.c_void_p * 1)(66)
    def squares(t=tensor, n=1, d=0, total=64, ws=64, size=1 << 20):
        return lib.bcclGradSquares(t, one, n, d, 0, p(total), p(ws), size, None)
    refused(squares(n=-1), "tensor list")
    refused(squares(t=None), "tensor list")
    refused(squares(d=1), "dtype")
    refused(squares(t=odd), "misaligned")
    refused(squares(total=0), "sum")
    refused(squares(total=68), "sum")
    refused(squares(ws=0), "workspace")
    refused(squares(size=8), "workspace")
    refused(lib.bcclGradClip(tensor, tensor, one, 1, 4, 0, p(64), 1.0, 0.0, None, None), "in place")
    refused(lib.bcclGradClip(tensor, tensor, one, 1, 0, 4, p(64), 1.0, 0.0, None, None), "dtypes")
    refused(lib.bcclGradClip(tensor, tensor, one, 1, 0, 0, p(64), -1.0, 0.0, None, None), "max_norm")
    refused(lib.bcclGradClip(tensor, tensor, one, 1, 0, 0, p(64), float("nan"), 0.0, None, None), "max_norm")

    def fwd(kind=0, x=64, xs=8, w=64, b=64, y=64, ys=8, mean=64, rstd=64, rows=2, h=8, eps=1e-5, d=0, wd=0):
        return lib.bcclNormForward(kind, p(x), xs, p(w), p(b), p(y), ys, p(mean), p(rstd), rows, h, eps, d, wd, None)
    refused(fwd(kind=2), "kind")
    refused(fwd(kind=1), "bias")
    refused(fwd(d=2), "dtypes")
    refused(fwd(d=0, wd=4), "dtypes")
    refused(fwd(h=0), "shape")
    refused(fwd(h=(1 << 23) + 1), "shape")
    refused(fwd(rows=-1), "shape")
    refused(fwd(eps=-1.0), "eps")
    refused(fwd(x=0), "input")
    refused(fwd(x=66), "input")
    refused(fwd(ys=7), "input or output")
    refused(fwd(xs=-8), "input")
    refused(fwd(rstd=0), "statistics")
    refused(fwd(mean=0), "statistics")

    def bwd(ws=64, size=1 << 30, **k):
        a = dict(kind=0, dy=64, x=64, mean=64, rstd=64, w=64, dx=64, dxs=8, dw=64, db=64, rows=2, h=8, d=0, wd=0)
        a.update(k)
        return lib.bcclNormBackward(a["kind"], p(a["dy"]), 8, p(a["x"]), 8, p(a["mean"]), p(a["rstd"]), p(a["w"]), p(a["dx"]),
                                    a["dxs"], p(a["dw"]), p(a["db"]), a["rows"], a["h"], a["d"], a["wd"], p(ws), size, None)
    assert lib.bcclNormBackwardWorkspace(0, 2, 8, 0) > 0
    refused(bwd(size=lib.bcclNormBackwardWorkspace(0, 2, 8, 0) - 1), "workspace")
    refused(bwd(ws=0), "workspace")
    refused(bwd(ws=72), "workspace")
    refused(bwd(kind=1), "gradient")
    refused(bwd(dxs=4), "input or output")
    refused(bwd(dy=0), "input")

    def emb(ids=64, it=3, n=2, t=64, ts=8, rows=4, h=8, first=0, out=64, os=8, d=0):
        return lib.bcclEmbeddingForward(p(ids), it, n, p(t), ts, rows, h, first, 1.0, p(out), os, d, None)
    refused(emb(it=0), "dtypes")
    refused(emb(ids=0), "ids")
    refused(emb(ids=68), "ids")
    refused(emb(n=1 << 31), "shape")
    refused(emb(rows=(1 << 31) - 1), "shape")
    refused(emb(first=-1), "shape")
    refused(emb(t=0), "table")
    refused(emb(os=4), "output")

    def embb(size=1 << 40, **k):
        a = dict(n=2, rows=4, h=8, d=4, od=4, ws=64)
        a.update(k)
        return lib.bcclEmbeddingBackward(p(64), 8, p(64), 3, a["n"], p(64), a["rows"], a["h"], 0, 1.0, 0, 0, 0, a["d"], a["od"],
                                         p(a["ws"]), size, None)
    refused(embb(size=lib.bcclEmbeddingBackwardWorkspace(2, 4, 8) - 1), "workspace")
    refused(embb(od=5), "dtypes")
    refused(embb(n=-1), "shape")

    def sort(tokens=4, top=2, experts=8, slots=64, ws=64, size=1 << 30):
        return lib.bcclExpertSort(p(64), 2, tokens, top, experts, p(slots), p(64), p(64), p(ws), size, None)
    refused(sort(top=65), "shape")
    refused(sort(experts=1024), "shape")
    refused(sort(tokens=1 << 30), "shape")
    refused(sort(slots=0), "null")
    assert lib.bcclExpertSortWorkspace(4, 2) == 0
    refused(sort(tokens=1 << 20, size=lib.bcclExpertSortWorkspace(1 << 20, 2) - 1), "workspace")
    refused(sort(tokens=1 << 20, ws=0), "workspace")
    refused(lib.bcclExpertDispatch(p(64), 8, p(64), p(64), 4, 2, 8, 0, p(64), 0, None), "shape")
    refused(lib.bcclExpertDispatch(p(66), 8, p(64), p(64), 4, 2, 8, 8, p(64), 0, None), "misaligned")
    refused(lib.bcclExpertCombine(p(64), p(64), p(64), 4, 4, 2, 8, p(64), 8, 0, None), "dtypes")
    refused(lib.bcclExpertCombine(p(64), None, p(64), 0, 4, 2, 8, p(64), 8, 0, None), "null")
    refused(lib.bcclExpertCombineBackward(p(64), 8, p(0), p(64), p(64), p(64), 0, 4, 2, 8, 8, p(64), p(64), 0, None), "null")


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused(monkeypatch):
    """The guard's rule with stand-ins for the stream and the capture: the leaf's accumulation node was
    made on another stream and still lives."""
    from originccl_b200.ops import _capture
    leaf = torch.ones(3, requires_grad=True)

    class Op(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            _capture.guard("op", x)
            return x * 2

        @staticmethod
        def backward(ctx, g):
            return g * 2

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    held = Op.apply(leaf)                          # an eager graph, stream 0
    marks = torch.autograd.graph.get_gradient_edge(leaf).node.metadata
    assert marks[_capture._KEY] == 0
    marks[_capture._KEY] = 7                       # as if made on stream 7
    Op.apply(leaf)                              # fine while nothing is captured
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="still alive"):
        Op.apply(leaf)
    del held, marks
    Op.apply(leaf)                              # the eager graph is gone, and its node with it


def test_tensors_without_storage_are_refused():
    """A wrapper has shape, type, layout and device of its own but a null data pointer, which the C
    interface reads as "not given": it must not take the place of a weight that is then left out."""
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, inner):
            return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError(f"{func} must not run")

    x, w = torch.zeros(4, 8), torch.ones(8)
    ids = torch.zeros(4, 1, dtype=torch.int32)
    order = experts.ExpertOrder(ids, ids.reshape(-1), torch.zeros(3, dtype=torch.int32))
    bare = Wrapper(w)
    assert bare.is_contiguous() and bare.data_ptr() == 0
    for what, call in (("weight", lambda: norm.rms_norm_forward(x, bare)),
                       ("weight", lambda: norm.layer_norm_forward(x, bare, w)),
                       ("bias", lambda: norm.layer_norm_forward(x, w, bare)),
                       ("weight", lambda: norm.rms_norm_backward(x, x, torch.zeros(4), bare)),
                       ("out", lambda: norm.rms_norm_forward(x, w, out=Wrapper(x))),
                       ("input", lambda: norm.rms_norm_forward(Wrapper(x), w)),
                       ("weight", lambda: embedding.embedding_forward(ids, Wrapper(x))),
                       ("weights", lambda: experts.combine_forward(x, order, Wrapper(torch.ones(4, 1)))),
                       ("weights", lambda: experts.combine_backward(x, x, order, Wrapper(torch.ones(4, 1)))),
                       ("rows", lambda: experts.combine_forward(Wrapper(x), order)),
                       ("input", lambda: experts.dispatch_forward(Wrapper(x), order))):
        with pytest.raises(TypeError, match=f"{what} must have memory"):
            call()


def public_calls(leaf):
    """Every differentiable entry point with `leaf` [4, 8] or a slice of it among its inputs. On host tensors each
    ends at the check of the device, behind everything that is done before a kernel's call."""
    ids = torch.zeros(4, 1, dtype=torch.int32)
    order = experts.ExpertOrder(ids, ids.reshape(-1), torch.zeros(3, dtype=torch.int32))
    return (lambda: norm.rms_norm(leaf, None), lambda: norm.layer_norm(leaf, torch.ones(8), torch.ones(8)),
            lambda: embedding.embedding(ids, leaf), lambda: experts.dispatch(leaf, order), lambda: experts.combine(leaf, order),
            lambda: experts.combine(leaf, order, torch.ones(4, 1)))


@pytest.mark.parametrize("mode", [torch.inference_mode, torch.no_grad])
def test_the_capture_rule_holds_only_where_a_graph_is_recorded(monkeypatch, mode):
    """Serving: parameters that require gradients, and no graph. The calls get past the rule (host tensors
    are refused behind it) in every mode, also while something is captured beside an eager graph."""
    leaf = torch.ones(4, 8, requires_grad=True)
    for call in public_calls(leaf):
        with mode(), pytest.raises(ValueError, match="CUDA"):
            call()
    with torch.inference_mode(), torch.enable_grad(), pytest.raises(ValueError, match="CUDA"):
        norm.rms_norm(leaf, None)
    held = leaf * 2
    torch.autograd.graph.get_gradient_edge(leaf).node.metadata["bccl_stream"] = 7  # as if made on stream 7
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in public_calls(leaf):
        with mode(), pytest.raises(ValueError, match="CUDA"):
            call()
        with pytest.raises(RuntimeError, match="still alive"):
            call()
    del held


def test_the_capture_rule_knows_nodes_of_other_operators(monkeypatch):
    """The leaf's node was made by an operator that leaves no mark: its own stream counts (a stand-in here,
    host tensors have none)."""
    from originccl_b200.ops import _capture
    leaf = torch.ones(4, 8, requires_grad=True)
    assert _capture._ops.leaf_stream(leaf) is None
    held = leaf * 2
    assert _capture._ops.leaf_stream(leaf) is None and _capture._ops.leaf_stream(held) is None

    class Ops:
        leaf_stream = staticmethod(lambda t: 7)
    monkeypatch.setattr(_capture, "_ops", Ops)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    _capture.guard("op", leaf)  # fine while nothing is captured
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="still alive"):
        _capture.guard("op", leaf)


def test_gradients_without_storage_are_refused():
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, n):
            return torch.Tensor._make_wrapper_subclass(cls, (n,), dtype=torch.float32, device=torch.device("cuda", 0))

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError(f"{func} must not run")

    for call in (lambda: gradients.grad_norm([Wrapper(4)]), lambda: gradients.clip_grad_norm([Wrapper(4)], 1.0),
                 lambda: gradients.clip_grad_norm([Wrapper(4)], 1.0, outs=[Wrapper(4)])):
        with pytest.raises(TypeError, match="each gradient must have memory"):
            call()


def test_host_gradients_need_no_extension(monkeypatch):
    """Where the extension was not built (no CUDA headers of PyTorch), ranks with host tensors still clip."""
    import importlib

    def missing():
        raise ImportError("not built")
    monkeypatch.setattr(_native, "ops", missing)
    try:
        again = importlib.reload(gradients)
        g = [torch.full((4,), 3.0), torch.full((9,), 1.0)]
        assert abs(again.grad_norm(g).item() - 45.0 ** 0.5) <= 45.0 ** 0.5 * 2 ** -23
        again.clip_grad_norm(g, 1.0)
        assert abs(g[0][0].item() - 3.0 / 45.0 ** 0.5) <= 2 ** -20
        with pytest.raises(ValueError, match="no gradients"):
            again.grad_norm([])
    finally:
        monkeypatch.undo()
        importlib.reload(gradients)


def test_the_capture_rule_looks_at_nothing_without_a_capture(monkeypatch):
    """Eager training calls pay for no look-up of nodes."""
    from originccl_b200.ops import _capture

    def never(*_):
        raise AssertionError("looked up")
    monkeypatch.setattr(_capture, "guard", never)
    leaf = torch.ones(4, 8, requires_grad=True)
    for initialized in (False, True):
        monkeypatch.setattr(torch.cuda, "is_initialized", lambda: initialized)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        for call in public_calls(leaf):
            with pytest.raises(ValueError, match="CUDA"):
                call()


@pytest.mark.parametrize("dtype", [torch.float32, bf, torch.float16])
def test_a_native_stack_has_the_norms_of_torch(monkeypatch, dtype):
    """Small activations, where the epsilon that a norm without one of its own takes decides. The kernel's place
    is taken by the formula in 64 bits. The weights are ones, so each side rounds once: a step apart at most
    (float32 sums of 64 squares and the root: 70 more)."""
    from originccl_b200.models import TinyLlamaStack

    def rms_norm(x, weight, eps):
        d = x.double()
        return (d * (d.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double()).to(x.dtype)
    monkeypatch.setattr(norm, "rms_norm", rms_norm)
    x = (torch.randn(5, 64, generator=torch.Generator().manual_seed(1)) * 0.01).to(dtype)
    m = TinyLlamaStack(hidden=64, ffn=64, layers=1, dtype=dtype, native=True)
    for eps in (None, 1e-4):
        n = m.blocks[0]["norm"]
        n.eps = eps
        want = n(x).double()
        assert ((m._norm(n, x).double() - want).abs() <= (torch.finfo(dtype).eps + 70 * 2 ** -24) * want.abs() + 1e-7).all()


def test_host_clipping_refuses_outs_of_another_shape_or_type():
    """As on a GPU: a larger out took the clipped values broadcast, and a narrower type lost them."""
    g = [torch.ones(4), torch.ones(2, 3, dtype=bf)]
    fine = [torch.full((4,), 7.0), torch.full((2, 3), 7.0)]
    for i, out in ((0, torch.full((3, 4), 7.0)), (0, torch.full((4,), 7.0, dtype=bf)), (1, torch.full((2, 3), 7.0).half()),
                   (1, torch.full((5, 2, 3), 7.0)), (0, torch.full((4,), 7.0, dtype=torch.float64))):
        outs = list(fine)
        outs[i] = out
        with pytest.raises(ValueError, match="out|float32"):
            gradients.clip_grad_norm(g, 1.0, outs=outs)
        assert all((t == 7).all() for t in outs)
    gradients.clip_grad_norm(g, 10.0, outs=fine)
    assert all((t == 1).all() for t in fine)
