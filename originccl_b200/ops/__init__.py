"""Compute ops built on the library's sm_100a kernels: tensor-core GEMM, fused TP GEMM+collective, and
the operators of a step beside the collectives (gradient norm and clipping, norms, embedding, tokens
sorted by expert), which load the package's extension on first use."""
from . import gemm, tp  # noqa: F401

__all__ = ["embedding", "experts", "gemm", "gradients", "norm", "tp"]


def __getattr__(name):
    if name in __all__:
        import importlib
        return importlib.import_module("." + name, __name__)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
