"""RMSNorm and SwiGLU modules (tokserve/engine/layers.py).

Parameters, their names, shapes and creation order match the reference
modules, so a state dict moves between the two and a seeded random
initialisation produces the same weights. The forward passes run on HIP
tensors only: RMSNorm through the tks_rms_norm kernel (the reference's
rounding: normalised value rounded to the input dtype, then times the weight,
output dtype = promote(weight, input)), SwiGLU as one library GEMM over the
stacked gate/up weights, the tks_silu_mul kernel, and the down GEMM. MXFP4Linear
stands in for a projection whose weight is MXFP4 (this library's own addition): the
two GEMMs are then block-scaled products over rows quantized on the way.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.nn import functional

from tokserve_amd.kernels import ops

__all__ = ["MXFP4Linear", "RMSNorm", "SwiGLU", "fused_linear", "fused_weight"]


class RMSNorm(nn.Module):
    """Llama RMSNorm with a learned scale."""

    def __init__(self, hidden_size: int, *, epsilon: float = 1e-6) -> None:
        super().__init__()
        if hidden_size < 1:
            raise ValueError("hidden_size must be positive")
        if epsilon <= 0.0:
            raise ValueError("epsilon must be positive")
        self.hidden_size = hidden_size
        self.epsilon = epsilon
        self.weight = nn.Parameter(torch.ones(hidden_size))

    def forward(
        self, inputs: torch.Tensor, residual: torch.Tensor | None = None
    ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
        """weight * to_in(x * rsqrt(mean(x^2) + eps)); with `residual`, x = to_in(inputs +
        residual) is formed first and (normalised, x) returned."""

        if inputs.ndim < 1:
            raise ValueError("inputs must have at least one dimension")
        if inputs.shape[-1] != self.hidden_size:
            raise ValueError("inputs must use the configured hidden_size")
        if residual is None:
            return ops.rms_norm(inputs, self.weight, self.epsilon)
        summed = torch.empty_like(inputs)
        normalized = ops.rms_norm(inputs, self.weight, self.epsilon, residual=residual,
                                  residual_out=summed)
        return normalized, summed


class MXFP4Linear(nn.Module):
    """A bias-free projection with MXFP4 weights, in place of a bias-free nn.Linear.

    Buffers `codes` (out, in / 2) and `scales` (out, in / 32) hold the bytes of
    ops.mxfp4_quantize's results: as uint8, so that .to(dtype) leaves them alone.
    """

    def __init__(self, in_features: int, out_features: int, *,
                 device: torch.device | str | None = None) -> None:
        super().__init__()
        if in_features < 1 or in_features % ops.MXFP4_BLOCK:
            raise ValueError(f"in_features must be a positive multiple of {ops.MXFP4_BLOCK}")
        if out_features < 1:
            raise ValueError("out_features must be positive")
        self.in_features = in_features
        self.out_features = out_features
        self.register_buffer("codes", torch.zeros(out_features, in_features // 2,
                                                  dtype=torch.uint8, device=device))
        self.register_buffer("scales", torch.zeros(out_features, in_features // ops.MXFP4_BLOCK,
                                                   dtype=torch.uint8, device=device))

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> MXFP4Linear:
        """The weights of `linear` (on a HIP device, without a bias), each block quantized."""

        if linear.bias is not None:
            raise ValueError("MXFP4 projections have no bias")
        weight = linear.weight.detach()
        quantized = cls(linear.in_features, linear.out_features, device=weight.device)
        ops.mxfp4_quantize(weight, codes=quantized.codes.view(ops.MXFP4_DTYPE),
                           scales=quantized.scales.view(ops.MXFP4_SCALE_DTYPE))
        return quantized

    def forward(self, inputs: torch.Tensor) -> torch.Tensor:
        return ops.mxfp4_linear(inputs, self.codes.view(ops.MXFP4_DTYPE),
                                self.scales.view(ops.MXFP4_SCALE_DTYPE))

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}"


def fused_weight(owner: nn.Module, linears: list[nn.Module], cache_name: str,
                 name: str = "weight") -> torch.Tensor:
    """One matrix stacking the rows of the tensors `name` of `linears`, which then view into it.

    The first call (and any call after .to() or load_state_dict gave one of
    them new storage) concatenates them and rebinds the data of each to its
    row range of the result, so the fused matrix costs no extra memory and
    stays the modules' own storage.
    """

    fused = getattr(owner, cache_name, None)
    if fused is not None:
        offset = 0
        intact = True
        for linear in linears:
            tensor = getattr(linear, name)
            rows = tensor.shape[0]
            view = fused[offset : offset + rows]
            if (tensor.data_ptr() != view.data_ptr() or tensor.dtype != fused.dtype
                    or tensor.device != fused.device):
                intact = False
                break
            offset += rows
        if intact:
            return fused
    # Built outside inference mode, so the parameters stay ordinary tensors that
    # .to() and load_state_dict may later update in place.
    with torch.inference_mode(False), torch.no_grad():
        fused = torch.cat([getattr(linear, name).detach() for linear in linears],
                          dim=0).contiguous()
        offset = 0
        for linear in linears:
            tensor = getattr(linear, name)
            rows = tensor.shape[0]
            tensor.data = fused[offset : offset + rows]
            offset += rows
    object.__setattr__(owner, cache_name, fused)
    return fused


def fused_linear(owner: nn.Module, linears: list[nn.Module], cache_name: str,
                 inputs: torch.Tensor) -> torch.Tensor:
    """The projections `linears` (all nn.Linear or all MXFP4Linear) of the same inputs, side
    by side, as one product over their stacked rows."""

    if not isinstance(linears[0], MXFP4Linear):
        return functional.linear(inputs, fused_weight(owner, linears, cache_name))
    codes = fused_weight(owner, linears, cache_name + "_codes", "codes")
    scales = fused_weight(owner, linears, cache_name + "_scales", "scales")
    return ops.mxfp4_linear(inputs, codes.view(ops.MXFP4_DTYPE),
                            scales.view(ops.MXFP4_SCALE_DTYPE))


class SwiGLU(nn.Module):
    """Bias-free Llama SwiGLU feed-forward network."""

    def __init__(self, hidden_size: int, intermediate_size: int) -> None:
        super().__init__()
        if hidden_size < 1:
            raise ValueError("hidden_size must be positive")
        if intermediate_size < 1:
            raise ValueError("intermediate_size must be positive")
        self.hidden_size = hidden_size
        self.intermediate_size = intermediate_size
        self.gate_proj = nn.Linear(hidden_size, intermediate_size, bias=False)
        self.up_proj = nn.Linear(hidden_size, intermediate_size, bias=False)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, bias=False)

    def forward(self, inputs: torch.Tensor) -> torch.Tensor:
        """down(silu(gate(x)) * up(x))."""

        if inputs.ndim < 1:
            raise ValueError("inputs must have at least one dimension")
        if inputs.shape[-1] != self.hidden_size:
            raise ValueError("inputs must use the configured hidden_size")
        gate_up = fused_linear(self, [self.gate_proj, self.up_proj], "_gate_up", inputs)
        return self.down_proj(ops.silu_mul(gate_up))
