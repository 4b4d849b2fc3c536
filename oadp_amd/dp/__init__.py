"""Consumer side of the OAKE feature files: access layers + ``LoadCLIPFeatures``, and
the loss a detector's classifier takes from them: ``TopLogitsDistillation``."""
from .distill import TopLogitsDistillation
from .features import LoadCLIPFeatures, PackAccessLayer, PthAccessLayer, build_access_layer, pack

__all__ = ['LoadCLIPFeatures', 'PackAccessLayer', 'PthAccessLayer', 'TopLogitsDistillation', 'build_access_layer', 'pack']
