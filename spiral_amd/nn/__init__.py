from .evolve import EvolveGCNO, WeightGRU
from .gatconv import GATConv
from .graphconv import GraphConv
from .int8linear import Int8Linear
from .layernorm import LayerNorm
from .sageconv import SAGEConv
from .sgconv import SGConv

__all__ = ["GraphConv", "SGConv", "SAGEConv", "GATConv", "EvolveGCNO", "WeightGRU", "LayerNorm", "Int8Linear"]
