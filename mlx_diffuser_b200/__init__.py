"""B200-native (sm_100a) TRELLIS sparse-voxel path: the drop-in for mlx_diffuser's
``SparseTensor`` / ``build_neighbor_map`` / ``SparseConv3D`` / ``sparse_conv3d`` /
``sparse_downsample`` / ``sparse_upsample``, backed by ``libsparsevox.so``, and the operators of a
transformer block over the same rows: ``rms_norm``, ``linear`` and ``sparse_self_attention`` with a
learned relative position bias, ``block_norm`` at the borders between blocks, ``dropout``, and a mixture of
experts (``route``, ``expert_linear``)."""

from ._native import check_device_status
from .kernels.block_norm import block_norm
from .kernels.dropout import dropout
from .kernels.expert import ExpertRoutes, expert_linear, route
from .kernels.linear import linear
from .kernels.norm import rms_norm
from .kernels.sparse import sparse_conv3d
from .layers.sparse import (
    SparseConv3D,
    SparseTensor,
    build_neighbor_map,
    position_buckets,
    sparse_downsample,
    sparse_self_attention,
    sparse_upsample,
)

__all__ = [
    "ExpertRoutes",
    "SparseConv3D",
    "SparseTensor",
    "block_norm",
    "build_neighbor_map",
    "check_device_status",
    "dropout",
    "expert_linear",
    "linear",
    "position_buckets",
    "rms_norm",
    "route",
    "sparse_conv3d",
    "sparse_downsample",
    "sparse_self_attention",
    "sparse_upsample",
]
