"""brovisionml_b200 -- B200-native (sm_100a) DSINE refine ops.

The product is the CUDA library ``_lib/libbvml_dsine.so`` and its C ABI
(``include/bvml_dsine.h``). This package loads that library and mirrors the
reference's op interface (``brovisionml::dsine::ray_relu`` /
``angmf_propagate`` in include/brovisionml/dsine_ops.h:25-54, plus the
brotensor convex-upsample / L2-normalise / slice calls of
src/dsine_refine.cpp:277-292) for Python callers, with torch tensors as the
device-memory carrier. Beside it, libbvml_blocks.so (``include/bvml_blocks.h``) holds the
feed-forward operators over rows of features (``blocks.py``), loaded by their first call.
Every op runs in the CUDA library; there is no CPU or PyTorch fallback: importing the
package fails loudly when libbvml_dsine.so is missing, calling a feed-forward operator when
theirs is.

Errors raise ``RuntimeError`` carrying the library's message, worded like the
reference's exceptions ("dsine ops: ..." / "dsine cuda: ...").
"""
from __future__ import annotations

from ._capi import (BVML_F16, BVML_F32, LIB_PATH, abi_version, check, lib,  # noqa: F401
                    loaded_library)
from .ops import (angmf_propagate, conv2d_nhwc, convex_upsample, l2_normalize_nchw,  # noqa: F401
                  pack_conv_weight, ray_relu, refine, refine_workspace_bytes, slice2d)
from .blocks import (BLOCKS_LIB_PATH, blocks_status, gated_linear,  # noqa: F401
                     gated_linear_backward, linear, linear_backward, pack_weight_e4m3, rms_norm,
                     rms_norm_backward, rms_norm_e4m3)

__all__ = ["ray_relu", "angmf_propagate", "convex_upsample", "l2_normalize_nchw", "slice2d",
           "conv2d_nhwc", "pack_conv_weight",
           "rms_norm", "rms_norm_e4m3", "rms_norm_backward", "linear", "linear_backward",
           "gated_linear", "gated_linear_backward", "pack_weight_e4m3", "blocks_status",
           "BLOCKS_LIB_PATH", "refine", "refine_workspace_bytes", "lib", "abi_version", "loaded_library",
           "LIB_PATH", "BVML_F32", "BVML_F16"]
