"""MI355X-native (gfx950) FP8 hot path of shyampathak22/cinnamon.

``cinnamon_amd.kernels`` is the drop-in for the reference's ``kernels`` module;
``cinnamon_amd.layers`` holds the FP8 grouped-expert layer, ``cinnamon_amd.moe`` the experts' gate,
dispatch and combine, ``cinnamon_amd.rotary`` the rotary positions of queries and keys, and
``cinnamon_amd.lm_head`` the output projection with its cross entropy.  The native code is
libcinnamon_fp8.so (C ABI: include/cinnamon_fp8.h), built by ``cinnamon_amd._build``.
"""
from . import _lib  # noqa: F401

__all__ = ["kernels", "layers", "lm_head", "moe", "rotary"]
