from .conv import SparseConv, KernelMapCache
from .activations import ReLU, ReLU6, LeakyReLU
from .normalizations import BatchNorm
from .experts import ExpertBlock
from .fusion import fuse_epilogues

__all__ = ["SparseConv", "KernelMapCache", "ReLU", "ReLU6", "LeakyReLU", "BatchNorm", "ExpertBlock",
           "fuse_epilogues"]
