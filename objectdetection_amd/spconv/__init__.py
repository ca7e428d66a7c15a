"""Drop-in for the subset of the `spconv` 1.x python API the reference calls
(call sites second/pytorch/models/middle.py:4,64-93,98,127-128,145,199,206,
second/pytorch/models/resnet.py:1,10,22,32,69, second/builder/voxel_builder.py:3).

Everything here runs on hand-written gfx950 HIP kernels through liblcf.so; there is no CPU path.
Make it importable under the name ``spconv`` with ``objectdetection_amd.dropin.install()``.
"""
from . import ops, utils  # noqa: F401
from .conv import (SparseConv2d, SparseConv3d, SparseConvolution, SubMConv2d,  # noqa: F401
                   SubMConv3d)
from .modules import (RMSNorm, SparseModule, SparseSequential, ToDense,  # noqa: F401
                      is_spconv_module)
from .tensor import SparseConvTensor  # noqa: F401

__version__ = "1.1+lcf"
