from .conv import SparseConv, KernelMapCache
from .activations import ReLU, ReLU6, LeakyReLU
from .normalizations import BatchNorm
from .attention import AttentionBlock
from .experts import ExpertBlock
from .fusion import fuse_epilogues

__all__ = ["SparseConv", "KernelMapCache", "ReLU", "ReLU6", "LeakyReLU", "BatchNorm",
           "AttentionBlock", "ExpertBlock", "fuse_epilogues"]
