"""mpemu.module_wrappers -- nn.Module shells around functional ops so that quantisation hooks can
attach to them (reference mpemu/module_wrappers/{matmul,eltwise,aggregate,adasparse}.py).  No
kernels live here: the shells call the stock torch op, or one of mpemu.functional (GroupedMatmul,
GroupedLinear, ScaledEmbedding); their inputs/outputs are cast by the hooks."""
from .ops import (AddMatmul, BatchMatmul, EltwiseAdd, EltwiseDiv, EltwiseMul, GroupedLinear, GroupedMatmul, Matmul, Mean,
                  Norm, ScaledEmbedding, SparseConv2d, SparseLinear)
