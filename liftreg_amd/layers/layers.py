"""Network building blocks used by the configured model, with the reference's class names,
constructor arguments and state-dict keys (src/liftreg/layers/layers.py), running on the
HIP kernels, forward and backward (liftreg_amd.autograd): `loss.backward()` of the reference's training
step reaches the parameters through the HIP backward kernels, never through another backend."""
import math
import numbers

import torch
import torch.nn as nn

from .. import ops
from ..autograd import ConvBlockFn, LayerNormFn, LinearFn, NCCFn
from .._hip import NCC_SQUARED


class LayerNorm(nn.Module):
    """Layer norm over the trailing `normalized_shape` axes, with torch.nn.LayerNorm's arguments and state-dict keys, followed in
    the same pass by LeakyReLU(negative_slope) (1.0: none).  Input float32 or bfloat16, weight and bias float32."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, negative_slope=1.0):
        super().__init__()
        self.normalized_shape = (normalized_shape,) if isinstance(normalized_shape, numbers.Integral) else tuple(normalized_shape)
        if not self.normalized_shape or min(self.normalized_shape) < 1:
            raise ValueError(f"normalized_shape must name at least one axis of at least one element, got {normalized_shape}")
        self.eps, self.negative_slope = float(eps), float(negative_slope)
        self.weight = nn.Parameter(torch.ones(self.normalized_shape)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(self.normalized_shape)) if elementwise_affine and bias else None
        self.premasked_grad = False      # set by the model where the consumer applies the LeakyReLU's mask (autograd.LayerNormFn)

    def forward(self, x):
        n = len(self.normalized_shape)
        if tuple(x.shape[-n:]) != self.normalized_shape:
            raise ValueError(f"the input's trailing axes must be {self.normalized_shape}, got shape {tuple(x.shape)}")
        w, b = (None if t is None else t.reshape(-1) for t in (self.weight, self.bias))
        y = LayerNormFn.apply(x.reshape(x.shape[:-n] + (math.prod(self.normalized_shape),)) if n > 1 else x, w, b, self.eps, self.negative_slope, self.premasked_grad)
        return y.view(x.shape) if n > 1 else y


class convBlock(nn.Module):
    """Conv3d(k3) + LeakyReLU(0.2) (layers/layers.py:335-372) on the fp32 MFMA implicit GEMM.

    `in_layout`/`out_layout` select NCDHW (the reference's layout, default) or channels-last
    NDHWC for activations that stay inside the encoder.

    `layernorm`: Conv3d + layer norm over each voxel's channels + LeakyReLU, the last two in one pass (the reference's
    block offers a batch norm there, which a batch of 1-8 volumes cannot feed).
    """

    def __init__(self, in_channels, out_channels, kernel_size=3, stride=1, padding=1, bias=True,
                 batchnorm=False, residual=False, nonlinear=nn.LeakyReLU(0.2),
                 in_layout=ops.LAYOUT_NCDHW, out_layout=ops.LAYOUT_NCDHW, layernorm=False):
        super().__init__()
        if kernel_size != 3 or padding != 1 or batchnorm or residual:
            raise NotImplementedError("only the configuration the model uses is built: k3, p1, no BN/residual")
        self.conv = nn.Conv3d(in_channels, out_channels, kernel_size, stride=stride, padding=padding, bias=bias)
        self.bn = None
        self.nonlinear = nonlinear
        self.residual = None
        self.stride = stride
        self.in_layout, self.out_layout = in_layout, out_layout
        # backward chaining inside an encoder (set by the model, see autograd.ConvBlockFn)
        self.premasked_grad = False
        self.mask_input_slope = None
        if nonlinear is None:
            self._slope = 1.0
        elif isinstance(nonlinear, nn.LeakyReLU):
            self._slope = float(nonlinear.negative_slope)
        else:
            raise NotImplementedError("fused epilogue supports LeakyReLU or None")
        self.norm = None
        if layernorm:
            if out_layout not in (ops.LAYOUT_NCDHW, ops.LAYOUT_NDHWC):
                raise ValueError("layernorm: out_layout must be LAYOUT_NCDHW or LAYOUT_NDHWC (a voxel's channels in one row)")
            self.norm = LayerNorm(out_channels, negative_slope=self._slope)

    def forward(self, x, packed=None):
        if self.norm is not None:
            # the conv runs without activation and channels-last; its gradient is the one the norm hands back
            y = ConvBlockFn.apply(x, self.conv.weight, self.conv.bias, self.stride, self.in_layout, ops.LAYOUT_NDHWC, 1.0, packed, True,
                                  self.mask_input_slope)
            self.norm.premasked_grad = self.premasked_grad
            y = self.norm(y)
            return y.permute(0, 4, 1, 2, 3).contiguous() if self.out_layout == ops.LAYOUT_NCDHW else y
        # Training, chained blocks: a 16-channel block whose consumer applies this block's LeakyReLU mask in its data
        # gradient (premasked_grad) also writes that mask as one byte per channel quad; it travels to the consumer as an
        # attribute of the activation tensor (`_lr_sign4`) and replaces the consumer's re-read of the activation.
        mask_out = None
        x_sign4 = getattr(x, "_lr_sign4", None) if self.mask_input_slope is not None else None
        if (self.premasked_grad and torch.is_grad_enabled() and self.conv.weight.requires_grad and
                ops.conv3d_mask_supported(x, self.conv.weight, self.stride, self.in_layout, self.out_layout)):
            B, _, D, W, H = x.shape
            mask_out = torch.empty((B, D, W, H, self.conv.out_channels // 4), dtype=torch.uint8, device=x.device)
        y = ConvBlockFn.apply(x, self.conv.weight, self.conv.bias, self.stride, self.in_layout, self.out_layout,
                              self._slope, packed, self.premasked_grad, self.mask_input_slope, mask_out, x_sign4)
        if mask_out is not None:
            y._lr_sign4 = mask_out
        return y


class FullyConnectBlock(nn.Module):
    """Linear + LeakyReLU(0.2) (layers/layers.py:413-439); `layernorm`: Linear + layer norm over the features + LeakyReLU."""

    def __init__(self, in_channels, out_channels, bias=True, nonlinear=nn.LeakyReLU(0.2), layernorm=False):
        super().__init__()
        self.fc = nn.Linear(in_channels, out_channels, bias=bias)
        self.nonlinear = nonlinear
        if nonlinear is None:
            self._slope = 1.0
        elif isinstance(nonlinear, nn.LeakyReLU):
            self._slope = float(nonlinear.negative_slope)
        else:
            raise NotImplementedError("fused epilogue supports LeakyReLU or None")
        self.norm = LayerNorm(out_channels, negative_slope=self._slope) if layernorm else None

    def forward(self, x):
        if self.norm is not None:
            return self.norm(LinearFn.apply(x, self.fc.weight, self.fc.bias, 1.0))
        return LinearFn.apply(x, self.fc.weight, self.fc.bias, self._slope)


class NCCLoss(nn.Module):
    """Squared, per-channel NCC variant (layers/layers.py:238-255)."""

    def forward(self, x, y):
        return NCCFn.apply(x, y, NCC_SQUARED)


class GaussianSmoothing(nn.Module):
    """Holds the Gaussian kernel buffer the reference model registers but never applies
    (layers/layers.py:441-504; constructed at …Backproj.py:24) so that `state_dict()` carries
    the same `gaussian_smooth.weight` entry and reference checkpoints load strictly."""

    def __init__(self, channels, kernel_size, sigma, dim=2):
        super().__init__()
        if isinstance(kernel_size, numbers.Number):
            kernel_size = [kernel_size] * dim
        if isinstance(sigma, numbers.Number):
            sigma = [sigma] * dim
        grids = torch.meshgrid([torch.arange(s, dtype=torch.float32) for s in kernel_size], indexing="ij")
        kernel = torch.ones(())
        for size, std, g in zip(kernel_size, sigma, grids):
            kernel = kernel * (1 / (std * math.sqrt(2 * math.pi)) * torch.exp(-((g - (size - 1) / 2) / std) ** 2 / 2))
        kernel = kernel / torch.sum(kernel)
        self.register_buffer('weight', kernel.view(1, 1, *kernel.size()).repeat(channels, *[1] * (kernel.dim() + 1)))
        self.groups = channels

    def forward(self, input):
        raise NotImplementedError("unused by the configured model (never called in the reference either)")
