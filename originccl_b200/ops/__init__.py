"""Compute ops built on the library's sm_100a kernels: tensor-core GEMM, fused TP GEMM+collective, and
the operators of a step beside the collectives (gradient norm and clipping, norms, embedding, tokens
sorted by expert)."""
from . import embedding, experts, gemm, gradients, norm, tp  # noqa: F401

__all__ = ["embedding", "experts", "gemm", "gradients", "norm", "tp"]
