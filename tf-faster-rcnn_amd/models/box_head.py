"""Layers of the detection head, between ``RoIPooling`` and ``Decoder``.

The reference builds its head from Keras layers (``models/faster_rcnn.py:320-326``: ``TimeDistributed`` Flatten, Dense 4096
with relu, Dropout, Dense 4096 with relu, Dropout, and the two output Dense layers).  ``QuantizedDense`` serves such a Dense
layer in 8-bit floating point, ``Dropout`` and ``GroupNormalization`` train; constructors and ``get_config()`` keys follow the
Keras layers of the same names, ``call(inputs)`` takes one tensor.
"""

from __future__ import annotations

from typing import Any, Dict, List, Optional, Sequence

import torch

from .. import _lib
from ..utils import head_utils
from .faster_rcnn import Layer


def _assigned(held: Optional[torch.Tensor], value: torch.Tensor) -> torch.Tensor:
    """``value`` written into the tensor that a layer already holds, where it fits, so that optimisers and captured graphs built
    on that tensor go on with it; ``value`` itself otherwise."""
    if held is None or held.shape != value.shape or held.dtype != value.dtype or held.device != value.device:
        return value
    with torch.no_grad():
        if value.element_size() == 1:  # 8-bit floating point is copied as bytes
            held.view(torch.uint8).copy_(value.view(torch.uint8))
        else:
            held.copy_(value)
    return held


class QuantizedDense(Layer):
    """A Dense layer whose kernel is stored as e4m3 with a scale per 128 x 128 block, for inference.

    The weights are taken once, by ``set_weights`` (the kernel quantised, the bias copied); a call quantises its input (a scale
    per row and 128 columns) and multiplies.  Like the other inference layers it lets no gradient through: inputs that require
    one are refused.
    """

    def __init__(self, units: int, activation: Optional[str] = None, scale_dtype: torch.dtype = torch.float32,
                 out_dtype: torch.dtype = torch.bfloat16, **kwargs: Any) -> None:
        super().__init__(**kwargs)
        self.units = int(units)
        self.activation = activation
        self.scale_dtype = scale_dtype
        self.out_dtype = out_dtype
        self.kernel: Optional[torch.Tensor] = None
        self.kernel_scales: Optional[torch.Tensor] = None
        self.bias: Optional[torch.Tensor] = None

    def get_config(self) -> Dict[str, Any]:
        config = super().get_config()
        config.update({"units": self.units, "activation": self.activation, "scale_dtype": self.scale_dtype, "out_dtype": self.out_dtype})
        return config

    def set_weights(self, weights: Sequence[torch.Tensor]) -> None:
        """``[kernel (inputs, units)]`` or ``[kernel, bias (units,)]``, in the layout of a Keras Dense layer.

        Weights set again are written into the tensors that the layer has, if they fit: captured graphs then use them.
        """
        if len(weights) not in (1, 2):
            raise ValueError(f"expected [kernel] or [kernel, bias], got {len(weights)} arrays")
        kernel = torch.as_tensor(weights[0])
        if kernel.dim() != 2 or kernel.shape[1] != self.units:
            raise ValueError(f"kernel must be (inputs, {self.units}), got {tuple(kernel.shape)}")
        device = kernel.device if kernel.is_cuda else _lib.require_gpu()
        bias = None
        if len(weights) == 2:
            bias = _lib.device_tensor(weights[1], torch.float32, device).detach()
            if tuple(bias.shape) != (self.units,):
                raise ValueError(f"bias must be ({self.units},), got {tuple(bias.shape)}")
        with torch.inference_mode(False):  # tensors made in that mode could not be written again outside it
            rows = kernel.detach().to(device).t().contiguous()
            kernel, scales = head_utils.quantize_blocks(rows, block_rows=head_utils.BLOCK, scale_dtype=self.scale_dtype)
            self.kernel, self.kernel_scales = _assigned(self.kernel, kernel), _assigned(self.kernel_scales, scales)
            self.bias = None if bias is None else _assigned(self.bias, bias.clone())

    def call(self, inputs: torch.Tensor) -> torch.Tensor:
        """``(..., inputs)`` fp32, fp16 or bf16 -> ``(..., units)`` of ``out_dtype``."""
        if self.kernel is None:
            raise ValueError(f"{self.name} has no weights: call set_weights([kernel, bias]) first")
        x, scales = head_utils.quantize_blocks(inputs, scale_dtype=self.scale_dtype)
        return head_utils.scaled_matmul(x, scales, self.kernel, self.kernel_scales, bias=self.bias, activation=self.activation,
                                        out_dtype=self.out_dtype)


class GroupNormalization(Layer):
    """Group normalisation over the last axis' channels, with an activation.

    ``gamma`` and ``beta`` start as ones and zeros of the first input's channels; they are fp32 tensors that may require
    gradients (``trainable``).  A first call without ``set_weights`` makes them and may not itself be captured.
    """

    def __init__(self, groups: int = 32, epsilon: float = 1e-3, activation: Optional[str] = None, **kwargs: Any) -> None:
        super().__init__(**kwargs)
        self.groups = int(groups)
        self.epsilon = float(epsilon)
        self.activation = activation
        self.gamma: Optional[torch.Tensor] = None
        self.beta: Optional[torch.Tensor] = None

    def get_config(self) -> Dict[str, Any]:
        config = super().get_config()
        config.update({"groups": self.groups, "epsilon": self.epsilon, "activation": self.activation})
        return config

    def set_weights(self, weights: Sequence[torch.Tensor]) -> None:
        """``[gamma (channels,), beta (channels,)]``; set again, they are written into the parameters that the layer has, if they
        fit: optimisers and captured steps built on those go on with them.
        """
        with torch.inference_mode(False):  # tensors made in that mode could not train later
            gamma, beta = (_lib.device_tensor(w, torch.float32).detach().clone() for w in weights)
            if gamma.dim() != 1 or gamma.shape != beta.shape:
                raise ValueError(f"gamma and beta must be (channels,), got {tuple(gamma.shape)} and {tuple(beta.shape)}")
            self.gamma = _assigned(self.gamma, gamma).requires_grad_(self.trainable)
            self.beta = _assigned(self.beta, beta).requires_grad_(self.trainable)

    def get_weights(self) -> List[torch.Tensor]:
        return [] if self.gamma is None else [self.gamma, self.beta]

    def call(self, inputs: torch.Tensor) -> torch.Tensor:
        """``(batch, ..., channels)`` -> the same shape and type."""
        if self.gamma is None:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{self.name}: call the layer once, or set its weights, before capturing it")
            channels, device = inputs.shape[-1], inputs.device if inputs.is_cuda else _lib.require_gpu()
            self.set_weights([torch.ones(channels, device=device), torch.zeros(channels, device=device)])
        return head_utils.group_norm(inputs, self.gamma, self.beta, self.groups, self.epsilon, self.activation)


class Dropout(Layer):
    """Dropout; every training call draws another mask from the layer's seed.

    The seed and the number of the call live in device memory and advance on the stream, so a captured training step draws
    anew at each replay.  The first training call on a device makes that memory and may not itself be captured.  Calls of one
    layer on several streams are for the caller to order, as with any tensor that a call updates.
    """

    def __init__(self, rate: float, seed: Optional[int] = None, **kwargs: Any) -> None:
        super().__init__(**kwargs)
        self.rate = float(rate)
        if not 0.0 <= self.rate < 1.0:
            raise ValueError(f"rate must be in [0, 1), got {rate}")
        self.seed = seed
        self._states: Dict[torch.device, torch.Tensor] = {}

    def get_config(self) -> Dict[str, Any]:
        config = super().get_config()
        config.update({"rate": self.rate, "seed": self.seed})
        return config

    def call(self, inputs: torch.Tensor, training: bool = False) -> torch.Tensor:
        """Any shape, fp32, fp16 or bf16; the input itself when not training or at rate 0."""
        if not training or self.rate == 0.0:
            return inputs
        inputs = head_utils._operand(inputs, "inputs")
        state = self._states.get(inputs.device)
        if state is None:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{self.name}: call the layer once before capturing it")
            seed = int(torch.randint(0, 2 ** 62, (1,)).item()) if self.seed is None else int(self.seed)
            seed = (seed + 2 ** 63) % 2 ** 64 - 2 ** 63  # the 64 bits as a signed integer
            with torch.inference_mode(False):  # a tensor made in that mode could not advance outside it
                state = self._states[inputs.device] = torch.tensor([seed, 0], dtype=torch.int64, device=inputs.device)
        used = state.clone()
        state[1:].add_(1)
        return head_utils.dropout(inputs, self.rate, used)
