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
wrong shapes, strides or devices ValueError. Nothing here synchronises or
keeps scratch, so calls can be captured into CUDA graphs. There is no backward
pass: tensors that require gradients are refused while gradients are enabled.
"""
from typing import NamedTuple, Optional

import torch

from . import _native

ACT_NONE, ACT_RELU, ACT_LEAKY_RELU = _native.ACT_NONE, _native.ACT_RELU, _native.ACT_LEAKY_RELU

_CODE = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16,
         torch.float8_e4m3fn: _native.E4M3}
_PLAIN = (torch.float32, torch.bfloat16, torch.float16)
TOP_MOST = 32


def _check(rc):
    if rc:
        _native.check(rc)


def _tensor(t, name, dtypes, device=None):
    """`t` as an input: a CUDA tensor of one of `dtypes`, on `device`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} is not one of "
                        f"{', '.join(str(d) for d in dtypes)}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor, got one on {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, but the call runs on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: requires a gradient, and this operator has no backward pass "
                         f"(use torch.no_grad())")


def _rows(t, name):
    """(rows, columns, row pitch) of a tensor seen as rows of its last dimension."""
    dims = t.dim()
    if dims == 2:
        m, n = t.shape
        ld, step = t.stride()
    elif dims == 1:
        m, n, ld, step = 1, t.shape[0], t.shape[0], t.stride(0)
    elif dims == 0:
        raise ValueError(f"{name}: expected at least one dimension")
    else:
        n = t.shape[-1]
        step = t.stride(-1)
        lead = [(s, d) for s, d in zip(t.shape[:-1], t.stride()[:-1]) if s != 1]
        m = 1
        for s, _ in lead:
            m *= s
        if m and any(outer[1] != inner[0] * inner[1] for outer, inner in zip(lead, lead[1:])):
            raise ValueError(f"{name}: the leading dimensions of shape {tuple(t.shape)} with "
                             f"strides {t.stride()} cannot be viewed as one")
        ld = lead[-1][1] if lead else n
    if m <= 1:
        ld = n
    if m and n and ((n > 1 and step != 1) or ld < n):
        raise ValueError(f"{name}: needs contiguous rows that do not overlap, got shape "
                         f"{tuple(t.shape)} with strides {t.stride()}")
    return m, n, max(ld, n)


def _vector(t, n, name):
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name}: expected shape ({n},), got {tuple(t.shape)}")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name}: needs contiguous elements")


def _out(out, shape, dtype, device, name):
    """`out`, or a new tensor of this shape."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _tensor(out, name, (dtype,), device)
    if out.shape != torch.Size(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(out.shape)}")
    return out


class _on:
    """Makes `device` the current one if it is not; gives its current stream."""

    __slots__ = ("index", "before")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def rms_norm(x, weight=None, *, residual=None, eps: float = 1e-6, quant: Optional[str] = None,
             group: int = 0, out=None, residual_out=None):
    """h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight, over rows.

    x: f32, bf16 or f16; residual: as x; weight: [columns], x's type or f32.
    Returns y in x's type or, with quant="e4m3", the codes (torch.float8_e4m3fn)
    and their f32 scales, one for each row (group 0) or each `group` (32, 64 or
    128) columns: y = codes * scales. With a residual, h in x's type comes
    last: y, h or codes, scales, h. h goes to `residual_out` (which may be x or
    residual itself) and y or the codes to `out` where these are given. y is
    computed from h before its rounding and rounded once."""
    _tensor(x, "x", _PLAIN)
    device, dtype = x.device, x.dtype
    m, n, ldx = _rows(x, "x")
    if quant is not None and quant != "e4m3":
        raise ValueError(f"quant: expected None or 'e4m3', got {quant!r}")
    if group not in (0, 32, 64, 128):
        raise ValueError(f"group: expected 0 (a row), 32, 64 or 128, got {group}")
    if group and quant is None:
        raise ValueError("group: only quantised outputs have groups")
    if not 0.0 < eps < float("inf"):
        raise ValueError(f"eps: must be positive and finite, got {eps}")
    w_ptr, w_code = None, 0
    if weight is not None:
        _tensor(weight, "weight", (dtype, torch.float32), device)
        _vector(weight, n, "weight")
        w_ptr, w_code = weight.data_ptr(), _CODE[weight.dtype]
    r_ptr = h_ptr = h = None
    ldr = ldh = 0
    if residual is not None:
        _tensor(residual, "residual", (dtype,), device)
        if residual.shape != x.shape:
            raise ValueError(f"residual: expected shape {tuple(x.shape)}, got "
                             f"{tuple(residual.shape)}")
        ldr = _rows(residual, "residual")[2]
        h = _out(residual_out, x.shape, dtype, device, "residual_out")
        ldh = _rows(h, "residual_out")[2]
        r_ptr, h_ptr = residual.data_ptr(), h.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out: given without a residual")
    y = _out(out, x.shape, torch.float8_e4m3fn if quant else dtype, device, "out")
    ldy = _rows(y, "out")[2]
    scales, s_ptr, lds = None, None, 0
    if quant:
        lds = (n + group - 1) // group if group else 1
        scales = torch.empty(x.shape[:-1] + (lds,), dtype=torch.float32, device=device)
        s_ptr = scales.data_ptr()
    code = _CODE[dtype]
    with _on(device) as stream:
        _check(_native.lib().b200_rms_norm(
            x.data_ptr(), ldx, r_ptr, ldr, code, w_ptr, w_code, eps, h_ptr, ldh, y.data_ptr(), ldy,
            _native.E4M3 if quant else code, s_ptr, lds, group, m, n, stream))
    if quant:
        return (y, scales) if h is None else (y, scales, h)
    return y if h is None else (y, h)


class W4Weights:
    """A [K, N] weight matrix in 4 bits, packed for dense_w4 (made by pack_w4
    or quantize_w4). `buffer` holds it; the other attributes say how."""

    def __init__(self, buffer, K, N, group, scale_dtype, has_zeros):
        self.buffer, self.K, self.N, self.group = buffer, K, N, group
        self.scale_dtype, self.has_zeros = scale_dtype, has_zeros

    @property
    def shape(self):
        return (self.K, self.N)

    @property
    def device(self):
        return self.buffer.device

    def dequantize(self):
        """The f32 matrix [K, N] that the packed weights stand for."""
        W = torch.empty((self.K, self.N), dtype=torch.float32, device=self.device)
        with _on(self.device) as stream:
            _check(_native.lib().b200_w4_dequantize(
                self.buffer.data_ptr(), _CODE[self.scale_dtype], int(self.has_zeros), self.K,
                self.N, self.group, W.data_ptr(), self.N, stream))
        return W


def _check_group(group):
    if group != 32 and (group <= 0 or group % 64):
        raise ValueError(f"group: expected 32 or a multiple of 64, got {group}")


def pack_w4(codes, scales, zeros=None, *, group: int = 128) -> W4Weights:
    """W[k, n] = scales[k // group, n] * (codes[k, n] - zeros[k // group, n]).

    codes: uint8 [K, N], 0..15; scales: f32, bf16 or f16 [ceil(K / group), N];
    zeros: uint8 of the scales' shape, 0..15 (8 where None)."""
    _check_group(group)
    _tensor(codes, "codes", (torch.uint8,))
    if codes.dim() != 2:
        raise ValueError(f"codes: expected two dimensions, got shape {tuple(codes.shape)}")
    K, N = codes.shape
    ldc = _rows(codes, "codes")[2]
    groups = (K + group - 1) // group
    held = {"scales": (scales, _PLAIN), "zeros": (zeros, (torch.uint8,))}
    pitch = {"zeros": 0}
    for name, (t, dtypes) in held.items():
        if t is None and name == "zeros":
            continue
        _tensor(t, name, dtypes, codes.device)
        if t.shape != (groups, N):
            raise ValueError(f"{name}: expected shape {(groups, N)}, got {tuple(t.shape)}")
        pitch[name] = _rows(t, name)[2]
    L = _native.lib()
    s_code = _CODE[scales.dtype]
    size = L.b200_w4_bytes(K, N, group, s_code, int(zeros is not None))
    if size < 0:
        _native.check_last()
    buffer = torch.empty(size, dtype=torch.uint8, device=codes.device)
    with _on(codes.device) as stream:
        _check(L.b200_w4_pack(codes.data_ptr(), ldc, scales.data_ptr(), pitch["scales"], s_code,
                              None if zeros is None else zeros.data_ptr(), pitch["zeros"], K, N,
                              group, buffer.data_ptr(), stream))
    return W4Weights(buffer, K, N, group, scales.dtype, zeros is not None)


def quantize_w4(W, *, group: int = 128, scale_dtype=torch.float32) -> W4Weights:
    """4-bit weights of the f32 matrix W [K, N]: scale = max|W| / 7 over each
    group of K and column (rounded to scale_dtype), code = round(W / scale) + 8."""
    _check_group(group)
    _tensor(W, "W", (torch.float32,))
    if W.dim() != 2:
        raise ValueError(f"W: expected two dimensions, got shape {tuple(W.shape)}")
    if scale_dtype not in _PLAIN:
        raise TypeError(f"scale_dtype: {scale_dtype} is not one of "
                        f"{', '.join(str(d) for d in _PLAIN)}")
    K, N = W.shape
    ldw = _rows(W, "W")[2]
    codes = torch.empty((K, N), dtype=torch.uint8, device=W.device)
    scales = torch.empty(((K + group - 1) // group, N), dtype=scale_dtype, device=W.device)
    with _on(W.device) as stream:
        _check(_native.lib().b200_w4_quantize(W.data_ptr(), ldw, K, N, group, codes.data_ptr(), N,
                                              scales.data_ptr(), N, _CODE[scale_dtype], stream))
    return pack_w4(codes, scales, group=group)


def dense_w4(x, w: W4Weights, bias=None, *, act: int = ACT_NONE, alpha: float = 0.0,
             x_scales=None, x_group: int = 0, out_dtype=None, out=None):
    """act(x @ W + bias) over rows of x [..., K], made for few rows (the weights
    are read once for each 64 rows, 21 in f32).

    x: f32, bf16, f16, or e4m3 codes with x_scales [..., 1] (x_group 0) or
    [..., ceil(K / x_group)] as rms_norm gives them. bias: [N], f32, bf16 or
    f16. The result has x's type, bf16 for e4m3, or out_dtype (f32, bf16,
    f16). Products are exact, sums run in f32, the result is rounded once."""
    if not isinstance(w, W4Weights):
        raise TypeError(f"w: expected W4Weights, got {type(w).__name__}")
    _tensor(x, "x", (torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn))
    device = x.device
    if w.device != device:
        raise ValueError(f"w: on {w.device}, but the call runs on {device}")
    m, k, ldx = _rows(x, "x")
    if k != w.K:
        raise ValueError(f"x: expected {w.K} columns, got {k}")
    if act not in (ACT_NONE, ACT_RELU, ACT_LEAKY_RELU):
        raise ValueError(f"act: unknown activation {act}")
    e4m3 = x.dtype == torch.float8_e4m3fn
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else torch.bfloat16 if e4m3 else x.dtype
    if out_dtype not in _PLAIN:
        raise TypeError(f"out_dtype: {out_dtype} is not one of "
                        f"{', '.join(str(d) for d in _PLAIN)}")
    s_ptr, lds = None, 0
    if x_scales is not None:
        if not e4m3:
            raise TypeError("x_scales: only an e4m3 x has scales")
        if x_group not in (0, 32, 64, 128):
            raise ValueError(f"x_group: expected 0 (a row), 32, 64 or 128, got {x_group}")
        _tensor(x_scales, "x_scales", (torch.float32,), device)
        shape = x.shape[:-1] + ((k + x_group - 1) // x_group if x_group else 1,)
        if x_scales.shape != shape:
            raise ValueError(f"x_scales: expected shape {tuple(shape)}, got "
                             f"{tuple(x_scales.shape)}")
        lds = _rows(x_scales, "x_scales")[2]
        s_ptr = x_scales.data_ptr()
    elif x_group:
        raise ValueError("x_group: given without x_scales")
    b_ptr, b_code = None, 0
    if bias is not None:
        _tensor(bias, "bias", _PLAIN, device)
        _vector(bias, w.N, "bias")
        b_ptr, b_code = bias.data_ptr(), _CODE[bias.dtype]
    y = _out(out, x.shape[:-1] + (w.N,), out_dtype, device, "out")
    ldy = _rows(y, "out")[2]
    with _on(device) as stream:
        _check(_native.lib().b200_dense_w4(
            x.data_ptr(), ldx, _CODE[x.dtype], s_ptr, lds, x_group, w.buffer.data_ptr(),
            _CODE[w.scale_dtype], int(w.has_zeros), w.group, b_ptr, b_code, y.data_ptr(), ldy,
            _CODE[out_dtype], m, w.N, k, act, alpha, stream))
    return y


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
    _tensor(logits, "logits", _PLAIN)
    device = logits.device
    t, v, ld = _rows(logits, "logits")
    lead = logits.shape[:-1]
    if not 0 <= top <= TOP_MOST:
        raise ValueError(f"top: expected 0 to {TOP_MOST}, got {top}")
    if top > v or (v == 0 and t):
        raise ValueError(f"top: {top} of {v} logits")
    tok_ptr = lp_ptr = lp = None
    if tokens is not None:
        _tensor(tokens, "tokens", (torch.int32,), device)
        if tokens.shape != lead:
            raise ValueError(f"tokens: expected shape {tuple(lead)}, got {tuple(tokens.shape)}")
        if not tokens.is_contiguous():
            raise ValueError("tokens: needs contiguous elements")
        lp = torch.empty(lead, dtype=torch.float32, device=device)
        tok_ptr, lp_ptr = tokens.data_ptr(), lp.data_ptr()
    entropy = torch.empty(lead, dtype=torch.float32, device=device)
    top_lp = top_tok = top_lp_ptr = top_tok_ptr = None
    if top:
        top_lp = torch.empty(lead + (top,), dtype=torch.float32, device=device)
        top_tok = torch.empty(lead + (top,), dtype=torch.int32, device=device)
        top_lp_ptr, top_tok_ptr = top_lp.data_ptr(), top_tok.data_ptr()
    with _on(device) as stream:
        _check(_native.lib().b200_token_logprobs(
            logits.data_ptr(), ld, _CODE[logits.dtype], t, v, tok_ptr, lp_ptr, entropy.data_ptr(),
            top, top_lp_ptr, top_tok_ptr, stream))
    return TokenLogprobs(lp, entropy, top_lp, top_tok)
