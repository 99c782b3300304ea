"""Module API of the tensor-product path (same class names as ``equitorch.nn``)."""
from . import functional  # noqa: F401
from .activations import Gate
from .cutoffs import CosineCutoff, MollifierCutoff, PolynomialCutoff
from .radials import BesselBasis
from .angular import SinCos
from .attention import GraphAttention
from .embedding import TypeEmbedding
from .gated import GatedLinear
from .graph_layers import SO3LinearGraph
from .linears import IrrepsLinear, IrrepWiseLinear, SO2Linear, SO3Linear
from .norm import MeanSquaredNorm, Norm, SquaredNorm
from .normalization import BatchRMSNorm, LayerRMSNorm
from .residual_norm import AddRMSNorm
from .sphericals import SphericalHarmonics
from .tensor_products import TensorDot, TensorProduct
from .type_loss import TypeCrossEntropy
from .wigner_d import DenseWignerRotation, SparseWignerRotation, WignerD
from .window import WindowAttention

__all__ = ["Gate", "MeanSquaredNorm", "Norm", "SquaredNorm", "BatchRMSNorm", "LayerRMSNorm", "SinCos", "IrrepsLinear", "IrrepWiseLinear", "SO2Linear", "SO3Linear", "SO3LinearGraph", "SphericalHarmonics",
           "TypeEmbedding", "GraphAttention", "GatedLinear", "AddRMSNorm", "WindowAttention", "TypeCrossEntropy",
           "TensorDot", "TensorProduct", "DenseWignerRotation", "SparseWignerRotation", "WignerD", "functional"]
