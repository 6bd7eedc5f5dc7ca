"""The CUDA operations of the engine: `kernels` (one function per entry point of
the compiled library), `int4` (weights and cache rows in 4 bits), `linear` (the choice of matrix product) and `library`
(building and loading).  Importing this package compiles nothing; the first
operation does."""
from . import int4, kernels
from .library import ExtensionError, KernelError, counters, lib, require_gpu
from .linear import glu_product, linear, per_head_linear, swiglu_product

__all__ = ["kernels", "int4", "linear", "per_head_linear", "swiglu_product", "glu_product", "lib", "require_gpu", "ExtensionError", "KernelError", "counters"]
