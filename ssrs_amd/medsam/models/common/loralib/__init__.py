"""loralib drop-in: the two layers MFNet uses (reference: medsam/models/common/loralib/layers.py), and PooledLinear: many adapters beside
one shared projection."""
from .....vit import Linear, LoRALayer, MergedLinear, PooledLinear  # noqa: F401
