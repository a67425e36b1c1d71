"""B200-native (sm_100a) Ozaki-scheme GEMM.

Drop-in for the ``ozaki_matmul`` path of WhFanatic/Ozaki_triton: the same
Python operator API (``ozaki_matmul``, ``split_matrix``, ``cross_gemm``,
``compute_split_bits``) backed by hand-written CUDA kernels in
``liboz_b200.so`` (C ABI: ``include/ozaki_b200.h``).

Beside it, the products of a mixture-of-experts layer: ``grouped_matmul`` and
its gradients, ``matmul_w4`` (4-bit weights) and ``orthogonalize``
(Newton-Schulz steps on the layer's updates); ``route``, ``dispatch`` and ``combine``
(the router with its balance loss, and the rows' way to the experts and back),
``fused_matmul`` (a product with bias, activation and residual) and
``clip_gradients`` (many gradients by their global norm), with their gradients.
"""

from .api import (  # noqa: F401
    INPUT_DTYPES,
    MAX_SPLITS,
    SLICE_DTYPE_INFO,
    compute_split_bits,
    cross_gemm,
    device_status,
    ozaki_matmul,
    ozaki_matmul_from_host,
    select_dot_accum_dtype,
    select_out_accum_dtype,
    slice_row_elems,
    split_matrix,
)
from .experts import (  # noqa: F401
    grouped_matmul,
    grouped_matmul_backward,
    matmul_w4,
    quantize_w4,
)
from .newton import orthogonalize  # noqa: F401
from .fused import fused_matmul, fused_matmul_backward  # noqa: F401
from .routing import (  # noqa: F401
    Routing,
    combine,
    combine_backward,
    dispatch,
    dispatch_backward,
    route,
    route_backward,
)
from .clipping import clip_gradients  # noqa: F401
from ._lib import OzakiError, OzakiLibraryError, load as load_library, version  # noqa: F401

__all__ = [
    "ozaki_matmul", "ozaki_matmul_from_host", "split_matrix", "cross_gemm", "compute_split_bits",
    "select_dot_accum_dtype", "select_out_accum_dtype", "slice_row_elems",
    "grouped_matmul", "grouped_matmul_backward", "matmul_w4", "quantize_w4", "orthogonalize",
    "fused_matmul", "fused_matmul_backward", "Routing", "route", "route_backward", "dispatch", "dispatch_backward",
    "combine", "combine_backward", "clip_gradients",
    "device_status", "OzakiError", "OzakiLibraryError", "load_library", "version",
]
