"""A detector's classifier learns from CLIP's answers on the crops whose embeddings the OAKE sweep stored.

The teacher's logits are cosines of a stored embedding (``clip_objects`` / ``clip_blocks`` of ``LoadCLIPFeatures``) with
the label embeddings of ``oadp_amd.prompts.vild``; what the student takes from them is the list of the ``top`` largest,
as log probabilities.  A list is ``top * 12`` bytes a crop, so it can be made once (``teacher``) and kept in place of the
embeddings, or made on the fly."""
from __future__ import annotations

import torch
import torch.nn.functional as F

from ..clip.logits import MAX_TOP, distill_top_logits, label_logits, token_logprobs


class TopLogitsDistillation:
    """``loss(student_logits, embeddings)`` -> KL(teacher || student) per crop, differentiable in the student's logits.

    ``labels`` [n, embed]: label embeddings on the student's device.  ``top`` (1 .. 128; at most n are there): entries of
    the teacher's list.  ``scale``: CLIP's logit scale; ``temperature`` T divides the teacher's and the student's logits
    alike, and the loss is multiplied by T^2 so that its gradient keeps its size.  ``tail``: what the list leaves out counts
    as one more outcome (``distill_top_logits``).  ``mask`` (bool [n]): the labels that are taught - the others are left out
    of the teacher's distribution (the student's is over all of them; with ``tail`` they share the bucket)."""

    def __init__(self, labels: torch.Tensor, *, top: int = 32, scale: float = 100.0, temperature: float = 1.0,
                 tail: bool = True, mask: torch.Tensor | None = None) -> None:
        if labels.dim() != 2 or labels.shape[0] < 1:
            raise ValueError(f'expected label embeddings [n >= 1, embed], got {tuple(labels.shape)}')
        if not 1 <= int(top) <= MAX_TOP:
            raise ValueError(f'top must be 1 .. {MAX_TOP}, got {top}')
        if not 0 < temperature < float('inf'):
            raise ValueError(f'temperature must be positive and finite, got {temperature}')
        if not 0 < scale / temperature <= 1e38:
            raise ValueError(f'scale / temperature must be positive and at most 1e38, got {scale} / {temperature}')
        if mask is not None and mask.dtype != torch.bool:
            raise TypeError(f'mask must be bool, got {mask.dtype}')
        if mask is not None and mask.shape != labels.shape[:1]:
            raise ValueError(f'expected a mask {(labels.shape[0],)}, got {tuple(mask.shape)}')
        self.labels = F.normalize(labels.detach().float(), dim=-1)
        self.mask = mask
        self.top = min(int(top), labels.shape[0])
        self.scale, self.temperature, self.tail = float(scale), float(temperature), bool(tail)

    @torch.no_grad()
    def teacher(self, embeddings: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(indices int64, log probabilities fp32) [..., top] of the crops' labels at the temperature."""
        answer = token_logprobs(label_logits(embeddings, self.labels), top=self.top, mask=self.mask,
                                scale=self.scale / self.temperature)
        return answer.top_indices, answer.top_logprobs

    def __call__(self, student_logits: torch.Tensor, embeddings: torch.Tensor | None = None, *,
                 teacher: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        """Loss [...] of student logits [..., n] against the crops' ``embeddings`` [..., embed] or a stored ``teacher``."""
        if (embeddings is None) == (teacher is None):
            raise ValueError('exactly one of embeddings and teacher is needed')
        if student_logits.shape[-1] != self.labels.shape[0]:
            raise ValueError(f'{self.labels.shape[0]} labels, student logits {tuple(student_logits.shape)}')
        indices, logprobs = self.teacher(embeddings) if teacher is None else teacher
        loss = distill_top_logits(student_logits, indices, logprobs, scale=1 / self.temperature, tail=self.tail)
        return loss if self.temperature == 1 else loss * self.temperature ** 2
