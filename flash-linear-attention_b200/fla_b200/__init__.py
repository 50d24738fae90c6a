# -*- coding: utf-8 -*-
"""fla_b200 — B200 (sm_100a) CUDA implementation of the chunked linear-attention hot path of
flash-linear-attention, behind the reference's `fla.ops` call signatures.

    from fla_b200.ops.gated_delta_rule import chunk_gated_delta_rule

`install_as_fla_ops()` registers the op modules under the names `fla.ops.<family>` so that code
written against the reference imports these kernels instead.
"""

import sys
import types

__version__ = "0.1.0"


def _replace(name, mod):
    """Put `mod` in the place of the module `name`. Names that `mod` does not have, and submodules, stay those of a module that was there."""
    there = sys.modules.get(name)
    if there is not None and there is not mod:
        def rest(attr):
            if hasattr(there, attr):
                return getattr(there, attr)
            raise AttributeError(f"module {name!r} has no attribute {attr!r}")

        mod.__getattr__ = rest
    sys.modules[name] = mod


def install_as_fla_ops():
    """Alias `fla.ops.{gla,simple_gla,retention,delta_rule,gated_delta_rule,hgrn}` to this package."""
    from . import ops
    from .ops import delta_rule, gated_delta_rule, gla, hgrn, retention, simple_gla
    root = sys.modules.get("fla")
    if root is None:
        root = types.ModuleType("fla")
        root.__path__ = []
        sys.modules["fla"] = root
    sys.modules["fla.ops"] = ops
    root.ops = ops
    for name, mod in (("gla", gla), ("simple_gla", simple_gla), ("retention", retention),
                      ("delta_rule", delta_rule), ("gated_delta_rule", gated_delta_rule), ("hgrn", hgrn)):
        _replace(f"fla.ops.{name}", mod)


def install_as_fla_modules():
    """Alias `fla.modules.{l2norm,fused_norm_gate,convolution,layernorm}` to this package's CUDA implementation."""
    from . import modules
    from .modules import convolution, fused_norm_gate, l2norm, layernorm
    root = sys.modules.get("fla")
    if root is None:
        root = types.ModuleType("fla")
        root.__path__ = []
        sys.modules["fla"] = root
    sys.modules["fla.modules"] = modules
    for name, mod in (("l2norm", l2norm), ("fused_norm_gate", fused_norm_gate), ("convolution", convolution), ("layernorm", layernorm)):
        _replace(f"fla.modules.{name}", mod)
    root.modules = modules
