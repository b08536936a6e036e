"""QAT-side use of the nearest-codeword kernel: the straight-through fake quantisation that the
reference's wrappers evaluate on every training step.

``fake_quant_weight`` (quant/dimq_wrapper.py:72-75, ``forward_mode == "hard_ste"``) computes
``weight + (hard_quantize_weight(weight, centers)[0] - weight).detach()``: forward value = the
hard-quantised weight (up to the rounding of the two additions), gradient = identity on the weight,
none on the centres (they learn through the DIMQ losses, quant/dimq.py:244-296).  The reference
builds a ``[chunk, K]`` distance matrix per chunk for that; here it is one pass over the weight in
the CUDA library.  The trainer, the losses and the wrapper classes themselves are outside this
backend's scope; this module is the drop-in for that one call.
"""

from __future__ import annotations

import torch

from . import _lib, ops


class _FakeQuantSTE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight: torch.Tensor, centers: torch.Tensor, group_rows):
        return ops.fake_quantize_ste(weight.detach(), centers.detach(), group_rows=group_rows)

    @staticmethod
    def backward(ctx, grad_out: torch.Tensor):
        return grad_out, None, None


def fake_quant_weight(weight: torch.Tensor, centers: torch.Tensor, chunk_size: int | None = None, *,
                      group_rows: int | None = None) -> torch.Tensor:
    """Straight-through hard quantisation of ``weight`` to its nearest centre.

    Same value and gradients as the reference expression
    ``weight + (hard_quantize_weight(weight, centers, chunk_size)[0] - weight).detach()``.
    ``chunk_size`` is accepted for signature compatibility (the kernel needs no chunking);
    ``centers`` may be ``[G, K]`` with ``group_rows`` rows of ``weight`` per codebook (additive).
    CUDA tensors only: there is no CPU path.
    """
    if centers.numel() == 0:
        raise ValueError("centers must be non-empty")
    return _FakeQuantSTE.apply(weight, centers, group_rows)


def fake_quant_activation(x: torch.Tensor, activation_centers: torch.Tensor, chunk_size: int | None = None) -> torch.Tensor:
    """``x + (q - x).detach()`` with ``q`` the nearest activation centre (quant/dimq_wrapper.py:80-85,
    without the running update of the centres, which belongs to the trainer)."""
    return _FakeQuantSTE.apply(x, activation_centers, None)


def mx_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
              checkpoint: str = "int8") -> torch.Tensor:
    """A linear layer that computes in microscaled 4-bit numbers and keeps its activations in 8 bits (or 4).

    Forward: ``q(x) @ q(weight).T + bias`` with ``q`` the rounding of ``ops.mx_quantize(., "fp4")``, fp32 sums, the result
    in ``x``'s type: what ``ops.mx_linear`` gives for the quantised weight.  Gradients go straight through ``q``:
    ``dx = grad @ q(weight)``, ``dweight = grad.T @ x8``, ``dbias = grad.sum(0)``, each in the type of what it belongs to.
    ``x8`` is the copy of ``x`` that is kept from forward to backward, ``mx_quantize(x, checkpoint)``: a little over one
    byte a value with ``"int8"``, or the forward's own ``q(x)`` at half a byte with ``"fp4"``.  Neither ``x`` nor
    ``weight`` is kept.  fp32, fp16 or bf16 CUDA tensors; the three may differ in type.

    It can be differentiated once.  A backward pass can be captured into a CUDA graph, as long as no eager autograd graph of the same leaves is still
    alive: PyTorch would synchronise with that graph's stream, which invalidates the capture.
    """
    return _lib.host().mx_layer(x, weight, bias, ops._mx_format(checkpoint))
