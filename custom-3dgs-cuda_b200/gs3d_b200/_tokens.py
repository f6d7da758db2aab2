"""The native torch side of the token operators (csrc/token_binding.cpp), bound to the entry points
of the library that custom_rasterizer_cuda has loaded. It never falls back to anything: if the
module is not built, importing it raises."""

from __future__ import annotations

import ctypes

import torch  # noqa: F401  (the module links against torch's libraries)

from custom_rasterizer_cuda import _lib

try:
    from . import _native as native
except ImportError as e:
    raise ImportError("gs3d_b200/_native.so is not built or does not match this torch; run "
                      "`python custom-3dgs-cuda_b200/build.py` (or __graft_entry__.build()) first"
                      ) from e

native.bind({name: ctypes.cast(getattr(_lib.lib, name), ctypes.c_void_p).value
             for name in ("gs_last_error", "gs_rotary_axes", "gs_rms_norm_forward",
                          "gs_rms_norm_e4m3", "gs_rms_norm_backward_workspace_size",
                          "gs_rms_norm_backward", "gs_cross_attention_workspace_size",
                          "gs_cross_attention_forward",
                          "gs_cross_attention_backward_workspace_size",
                          "gs_cross_attention_backward")})
