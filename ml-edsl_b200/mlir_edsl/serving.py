"""Serving a dense network token by token, on torch CUDA tensors.

The operators around the dense layers of a network whose weights are kept in
4 bits, through the C-ABI on the current stream of the tensors' device:

    rms_norm        norm of a layer's input with the residual's addition,
                    in the input's type or in 8 bits with scales
    quantize_w4, pack_w4 -> W4Weights
                    4-bit weights with a scale for each group of K
    dense_w4        act(X @ W + b) of few rows with such weights
    token_logprobs  log probabilities of given tokens, entropy and the most
                    probable tokens of rows of logits

    h_q, s, h = rms_norm(x, w, residual=h, quant="e4m3")
    logits = dense_w4(h_q, head, x_scales=s)
    scores = token_logprobs(logits, tokens, top=5)

Rows are the last dimension: tensors of any number of dimensions whose leading
ones can be viewed as one, with contiguous rows. Wrong types raise TypeError,
wrong shapes, strides or devices ValueError. Nothing here (but check) synchronises
or keeps scratch, so calls can be captured into CUDA graphs. There is no backward
pass: tensors that require gradients are refused while gradients are enabled, and
tensors with tangents of forward differentiation always.

dense_w4 of more than 8 rows (f32: 2) bounds the waits inside its kernel. One that
runs out, which no sound GPU lets happen, makes the results around it NaN;
check() raises it.
"""
import os
from importlib.machinery import ExtensionFileLoader
from importlib.util import module_from_spec, spec_from_file_location
from typing import NamedTuple, Optional

import torch

from . import _native

ACT_NONE, ACT_RELU, ACT_LEAKY_RELU = _native.ACT_NONE, _native.ACT_RELU, _native.ACT_LEAKY_RELU


def _load():
    """The module that checks arguments, makes outputs and calls the library
    (csrc/torch_calls.cpp). There is no fallback, as for the library."""
    path = os.path.join(os.path.dirname(_native.LIB_PATH), "b200torch.so")
    if not os.path.exists(path):
        raise RuntimeError(f"B200 torch module not found at {path}; build it with "
                           "`python ml-edsl_b200/build.py` (there is no fallback)")
    spec = spec_from_file_location("b200torch", path, loader=ExtensionFileLoader("b200torch", path))
    module = module_from_spec(spec)
    spec.loader.exec_module(module)
    module.set_errors(_native.B200Error, torch.OutOfMemoryError)
    return module


_calls = _load()


def rms_norm(x, weight=None, *, residual=None, eps: float = 1e-6, quant: Optional[str] = None,
             group: int = 0, out=None, residual_out=None):
    """h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight, over rows.

    x: f32, bf16 or f16; residual: as x; weight: [columns], x's type or f32.
    Returns y in x's type or, with quant="e4m3", the codes (torch.float8_e4m3fn)
    and their f32 scales, one for each row (group 0) or each `group` (32, 64 or
    128) columns: y = codes * scales. With a residual, h in x's type comes
    last: y, h or codes, scales, h. h goes to `residual_out` and y or the codes to
    `out` where these are given; h and y may take the place of x or of residual,
    but outputs that overlap anything else are refused. y is computed from h
    before its rounding and rounded once."""
    return _calls.rms_norm(x, weight, residual, eps, quant, group, out, residual_out)


class W4Weights:
    """A [K, N] weight matrix in 4 bits, packed for dense_w4 (made by pack_w4
    or quantize_w4). `buffer` holds it; the other attributes say how."""

    __slots__ = ("_packed",)

    def __init__(self, buffer, K, N, group, scale_dtype, has_zeros):
        self._packed = (buffer, K, N, group, scale_dtype, has_zeros)

    buffer = property(lambda self: self._packed[0])
    K = property(lambda self: self._packed[1])
    N = property(lambda self: self._packed[2])
    group = property(lambda self: self._packed[3])
    scale_dtype = property(lambda self: self._packed[4])
    has_zeros = property(lambda self: self._packed[5])
    shape = property(lambda self: self._packed[1:3])
    device = property(lambda self: self._packed[0].device)

    def dequantize(self):
        """The f32 matrix [K, N] that the packed weights stand for."""
        return _calls.dequantize_w4(self._packed)


def pack_w4(codes, scales, zeros=None, *, group: int = 128) -> W4Weights:
    """W[k, n] = scales[k // group, n] * (codes[k, n] - zeros[k // group, n]).

    codes: uint8 [K, N], 0..15; scales: f32, bf16 or f16 [ceil(K / group), N];
    zeros: uint8 of the scales' shape, 0..15 (8 where None)."""
    buffer = _calls.pack_w4(codes, scales, zeros, group)
    return W4Weights(buffer, codes.shape[0], codes.shape[1], group, scales.dtype,
                     zeros is not None)


def quantize_w4(W, *, group: int = 128, scale_dtype=torch.float32) -> W4Weights:
    """4-bit weights of the f32 matrix W [K, N]: scale = max|W| / 7 over each
    group of K and column (rounded to scale_dtype), code = round(W / scale) + 8. A
    group that holds an infinity or NaN, or whose scale is past scale_dtype's
    range, becomes NaN."""
    codes, scales = _calls.quantize_w4(W, group, scale_dtype)
    return pack_w4(codes, scales, group=group)


def dense_w4(x, w: W4Weights, bias=None, *, act: int = ACT_NONE, alpha: float = 0.0,
             x_scales=None, x_group: int = 0, out_dtype=None, out=None):
    """act(x @ W + bias) over rows of x [..., K], made for few rows: the weights
    are read once for each 128 rows (64 with groups of 32, a third of that in
    f32). From about 256 f32 rows the dense layer of the expanded weights is
    faster.

    x: f32, bf16, f16, or e4m3 codes with x_scales [..., 1] (x_group 0) or
    [..., ceil(K / x_group)] as rms_norm gives them. bias: [N], f32, bf16 or
    f16. The result has x's type, bf16 for e4m3, or out_dtype (f32, bf16,
    f16); it goes to `out` where that is given, which must not overlap an input.
    Products are exact, sums run in f32, the result is rounded once."""
    if not isinstance(w, W4Weights):
        raise TypeError(f"w: expected W4Weights, got {type(w).__name__}")
    return _calls.dense_w4(x, w._packed, bias, act, alpha, x_scales, x_group, out_dtype, out)


def check(device=None):
    """Waits for the current stream of `device` (the current one where None) and
    raises B200Error if a kernel there gave up a wait since the last check."""
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream().cuda_stream
        _native.check(_native.lib().b200_stream_sync(stream))


class TokenLogprobs(NamedTuple):
    """What token_logprobs gives; None where it was not asked for."""
    logprobs: Optional[torch.Tensor]      # f32 [...]
    entropy: torch.Tensor                 # f32 [...]
    top_logprobs: Optional[torch.Tensor]  # f32 [..., top]
    top_tokens: Optional[torch.Tensor]    # i32 [..., top]


def token_logprobs(logits, tokens=None, *, top: int = 0) -> TokenLogprobs:
    """Over rows of logits [..., V] (f32, bf16 or f16): log softmax at `tokens`
    (i32 [...]; 0 for negative ones, which mark padded rows, NaN for those past
    V), the entropy, and the `top` (0 to 32) most probable tokens with their
    log probabilities, the lowest index first among equals. Logits of -inf are
    masked; a row of nothing else gives -inf everywhere and an entropy of 0."""
    return tuple.__new__(TokenLogprobs, _calls.token_logprobs(logits, tokens, top))
