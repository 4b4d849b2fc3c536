"""Drop-in for the slice of the ``clip`` package (LutingWang/CLIP fork, reference README.md:44)
that OADP's OAKE path touches: ``load_default`` -> (model, preprocess), ``model.encode_image``,
``model.visual(objects, masks)``, ``model.dtype``, ``model.visual.grid``.  Beside it, operators on
logits (``clip.logits``): ``token_logprobs``, ``distill_top_logits``; ``CLIP.classify`` answers with them."""
from . import logits, model
from .logits import TokenLogprobs, distill_top_logits, label_logits, token_logprobs
from .model import CLIP, VisionTransformer, load, load_default
from .preprocess import Preprocess
from .settings import settings

__all__ = ['logits', 'model', 'CLIP', 'VisionTransformer', 'load', 'load_default', 'Preprocess', 'settings',
           'TokenLogprobs', 'distill_top_logits', 'label_logits', 'token_logprobs']
