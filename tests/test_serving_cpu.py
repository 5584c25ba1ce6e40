"""The serving operators without a GPU: what the C-ABI and the Python calls
refuse before anything is launched."""
import ctypes

import pytest
import torch

from mlir_edsl import _native, serving

INVALID, TOO_LARGE = 1, 7
BUF = ctypes.create_string_buffer(1 << 16)
P = ctypes.addressof(BUF) + (-ctypes.addressof(BUF)) % 256  # never read: the calls are refused
F32, BF16, F16, E4M3 = _native.F32, _native.BF16, _native.F16, _native.E4M3


def call(name, defaults, **change):
    args = dict(defaults, **change)
    rc = getattr(_native.lib(), name)(*args.values())
    return rc, _native.lib().b200_last_error().decode()


NORM = dict(X=P, ldx=64, R=P, ldr=64, dtype=BF16, w=P, w_dtype=BF16, eps=1e-6, H=P, ldh=64, Y=P,
            ldy=64, y_dtype=BF16, scales=None, lds=0, group=0, M=4, N=64, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(M=-1), "negative"), (dict(N=-1), "negative"), (dict(dtype=E4M3), "X must be"),
    (dict(dtype=9), "X must be"), (dict(w_dtype=F16), "w must be"), (dict(eps=0.0), "eps"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(y_dtype=F32), "Y must be"), (dict(y_dtype=E4M3), "needs scales"),
    (dict(scales=P), "needs scales"), (dict(group=64), "groups"),
    (dict(group=48, y_dtype=E4M3, scales=P), "group must be"),
    (dict(group=-32, y_dtype=E4M3, scales=P), "group must be"),
    (dict(X=None), "null"), (dict(Y=None), "null"), (dict(ldx=63), "pitch"),
    (dict(ldr=63), "pitch"), (dict(ldh=63), "pitch"), (dict(ldy=63), "pitch"),
    (dict(group=32, y_dtype=E4M3, scales=P, lds=1), "pitch of scales"),
    (dict(y_dtype=E4M3, scales=P, lds=0), "pitch of scales"),
    (dict(X=P + 1), "aligned"), (dict(R=P + 1), "aligned"), (dict(w=P + 1), "aligned"),
    (dict(H=P + 1), "aligned"), (dict(Y=P + 1), "aligned"),
])
def test_norm_refusals(change, text):
    rc, message = call("b200_rms_norm", NORM, **change)
    assert rc == INVALID and text in message, message


def test_norm_sizes():
    assert call("b200_rms_norm", NORM, M=0)[0] == 0
    assert call("b200_rms_norm", NORM, N=0)[0] == 0
    assert call("b200_rms_norm", NORM, M=1 << 31)[0] == TOO_LARGE


W4 = dict(X=P, ldx=128, x_dtype=BF16, x_scales=None, ldxs=0, x_group=0, packed=P, s_dtype=BF16,
          has_zeros=0, group=128, b=P, b_dtype=BF16, Y=P, ldy=64, y_dtype=BF16, M=2, N=64, K=128,
          act=0, alpha=0.0, stream=None)
SCALED = dict(x_dtype=E4M3, x_scales=P, ldxs=4)


@pytest.mark.parametrize("change,text", [
    (dict(M=-1), "negative"), (dict(N=-1), "negative"), (dict(K=-1), "negative"),
    (dict(group=0), "group must"), (dict(group=48), "group must"), (dict(group=96), "group must"),
    (dict(group=-64), "group must"), (dict(s_dtype=E4M3), "scales must"),
    (dict(act=3), "activation"), (dict(act=-1), "activation"), (dict(x_dtype=5), "X must"),
    (dict(y_dtype=E4M3), "Y must"), (dict(b_dtype=E4M3), "b must"),
    (dict(x_scales=P, ldxs=1), "only an e4m3"), (dict(x_group=32), "without x_scales"),
    (dict(SCALED, x_group=16), "x_group must"), (dict(SCALED, x_group=32, ldxs=3), "pitch of"),
    (dict(SCALED, ldxs=0), "pitch of"), (dict(X=None), "null"), (dict(packed=None), "null"),
    (dict(Y=None), "null"), (dict(ldx=127), "pitch"), (dict(ldy=63), "pitch"),
    (dict(packed=P + 8), "16-byte"), (dict(X=P + 1), "aligned"), (dict(Y=P + 1), "aligned"),
    (dict(b=P + 1), "aligned"), (dict(K=1 << 31), "range"), (dict(N=1 << 31), "range"),
])
def test_dense_w4_refusals(change, text):
    rc, message = call("b200_dense_w4", W4, **change)
    assert rc == INVALID and text in message, message


def test_dense_w4_nothing_to_do():
    assert call("b200_dense_w4", W4, M=0)[0] == 0
    assert call("b200_dense_w4", W4, N=0)[0] == 0


def test_w4_sizes():
    L = _native.lib()
    # strips of 64 columns by blocks of 64 of K: 2048 bytes each, then scales
    # and zeros of whole strips, each on a multiple of 256 bytes
    assert L.b200_w4_bytes(128, 64, 128, F16, 0) == 2 * 2048 + 256
    assert L.b200_w4_bytes(128, 64, 128, F32, 0) == 2 * 2048 + 256
    assert L.b200_w4_bytes(1001, 999, 32, F32, 1) == 16 * 16 * 2048 + 16 * 32 * 64 * 5
    assert L.b200_w4_bytes(0, 64, 128, F16, 1) == 0
    assert L.b200_w4_bytes(64, 64, 33, F16, 0) == -1
    assert "group" in L.b200_last_error().decode()


QUANT = dict(W=P, ldw=64, K=128, N=64, group=128, codes=P, ldc=64, scales=P, lds=64, s_dtype=F16,
             stream=None)
PACK = dict(codes=P, ldc=64, scales=P, lds=64, s_dtype=F16, zeros=P, ldz=64, K=128, N=64,
            group=128, packed=P, stream=None)
BACK = dict(packed=P, s_dtype=F16, has_zeros=0, K=128, N=64, group=128, W=P, ldw=64, stream=None)


@pytest.mark.parametrize("name,defaults,change", [
    ("b200_w4_quantize", QUANT, dict(W=None)), ("b200_w4_quantize", QUANT, dict(codes=None)),
    ("b200_w4_quantize", QUANT, dict(scales=None)), ("b200_w4_quantize", QUANT, dict(ldw=63)),
    ("b200_w4_quantize", QUANT, dict(ldc=63)), ("b200_w4_quantize", QUANT, dict(lds=63)),
    ("b200_w4_quantize", QUANT, dict(group=33)), ("b200_w4_quantize", QUANT, dict(W=P + 2)),
    ("b200_w4_quantize", QUANT, dict(s_dtype=3)), ("b200_w4_pack", PACK, dict(codes=None)),
    ("b200_w4_pack", PACK, dict(scales=None)), ("b200_w4_pack", PACK, dict(packed=None)),
    ("b200_w4_pack", PACK, dict(packed=P + 4)), ("b200_w4_pack", PACK, dict(ldz=63)),
    ("b200_w4_pack", PACK, dict(lds=63)), ("b200_w4_pack", PACK, dict(scales=P + 1)),
    ("b200_w4_pack", PACK, dict(K=-1)), ("b200_w4_dequantize", BACK, dict(packed=None)),
    ("b200_w4_dequantize", BACK, dict(W=None)), ("b200_w4_dequantize", BACK, dict(ldw=63)),
    ("b200_w4_dequantize", BACK, dict(packed=P + 4)), ("b200_w4_dequantize", BACK, dict(W=P + 2)),
])
def test_w4_refusals(name, defaults, change):
    rc, message = call(name, defaults, **change)
    assert rc == INVALID and message


TOKENS = dict(logits=P, ld=100, dtype=F32, T=3, V=100, tokens=P, logprobs=P, entropy=P, top=5,
              top_logprobs=P, top_tokens=P, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(T=-1), "negative"), (dict(V=-1), "negative"), (dict(dtype=E4M3), "logits must"),
    (dict(top=-1), "top must"), (dict(top=33), "top must"), (dict(V=4), "top exceeds"),
    (dict(V=0, top=0), "without logits"), (dict(tokens=None), "go with"),
    (dict(logprobs=None), "go with"), (dict(top_tokens=None), "null"),
    (dict(top_logprobs=None), "null"), (dict(logits=None), "null"), (dict(ld=99), "pitch"),
    (dict(logits=P + 2), "aligned"),
])
def test_token_logprobs_refusals(change, text):
    rc, message = call("b200_token_logprobs", TOKENS, **change)
    assert rc == INVALID and text in message, message


def test_token_logprobs_sizes():
    assert call("b200_token_logprobs", TOKENS, T=0)[0] == 0
    assert call("b200_token_logprobs", TOKENS, T=1 << 30)[0] == TOO_LARGE


def test_python_types_and_devices():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        serving.rms_norm(x)
    with pytest.raises(TypeError, match="dtype"):
        serving.rms_norm(x.double())
    with pytest.raises(TypeError, match="torch tensor"):
        serving.rms_norm([1.0])
    with pytest.raises(ValueError, match="CUDA tensor"):
        serving.token_logprobs(x)
    with pytest.raises(TypeError, match="dtype"):
        serving.token_logprobs(x.int())
    with pytest.raises(TypeError, match="W4Weights"):
        serving.dense_w4(x, x)
    with pytest.raises(ValueError, match="group"):
        serving.quantize_w4(x, group=40)
    with pytest.raises(TypeError, match="dtype"):
        serving.pack_w4(x, x)


def test_rows_of_tensors():
    rows = serving._calls.rows_of
    assert rows(torch.zeros(4, 6)) == (4, 6, 6)
    assert rows(torch.zeros(4, 8)[:, :6]) == (4, 6, 8)
    assert rows(torch.zeros(6)) == (1, 6, 6)
    assert rows(torch.zeros(2, 3, 6)) == (6, 6, 6)
    assert rows(torch.zeros(2, 3, 8)[..., :6]) == (6, 6, 8)
    assert rows(torch.zeros(2, 1, 6).transpose(0, 1)) == (2, 6, 6)
    assert rows(torch.zeros(5, 1)[:, :1]) == (5, 1, 1)
    assert rows(torch.zeros(1, 6).expand(1, 6)) == (1, 6, 6)
    assert rows(torch.zeros(0, 6)) == (0, 6, 6)
    for t in (torch.zeros(6, 4).t(), torch.zeros(4, 12)[:, ::2], torch.zeros(1, 6).expand(4, 6),
              torch.zeros(()), torch.zeros(3, 2, 6).transpose(0, 1),
              torch.zeros(1, 2, 6).expand(4, 2, 6)):
        with pytest.raises(ValueError):
            rows(t)


# ------------------------------------------------------------------- frontend
def _plan(fn):
    from mlir_edsl.functions import FunctionSignature, validate_function_body
    from mlir_edsl.lowering import lower
    sig = FunctionSignature.from_callable(fn)
    ast, _ = validate_function_body(fn, sig)
    return lower(ast, sig.param_names)


def test_frontend_steps():
    from mlir_edsl import Tensor, f32, i32, relu, rms_norm, token_logprobs

    def net(X: Tensor[f32, 3, 8], R: Tensor[f32, 3, 8], w: Tensor[f32, 8], W: Tensor[f32, 8, 5],
            b: Tensor[f32, 5], t: Tensor[i32, 3]) -> Tensor[f32, 3]:
        return token_logprobs(relu(rms_norm(X, w, R, eps=1e-5) @ W + b), t)
    plan = _plan(net)
    assert [s.op for s in plan.steps] == ["rms_norm_f32", "gemm_f32", "token_logprobs_f32"]
    norm, gemm, score = plan.steps
    assert [plan.params[r.index] for r in norm.inputs] == ["X", "w", "R"]
    assert norm.has_bias and norm.has_residual and norm.eps == 1e-5 and norm.shape == (3, 8)
    assert gemm.has_bias and score.shape == (3,)
    assert "rms_norm_f32(X, w, R, eps=1e-05) -> f32[3, 8]" in plan.describe()

    def bare(X: Tensor[f32, 3, 8], R: Tensor[f32, 3, 8]) -> Tensor[f32, 3, 8]:
        return rms_norm(X, residual=R)
    step = _plan(bare).steps[0]
    assert not step.has_bias and step.has_residual and step.eps == 1e-6


def test_frontend_refusals():
    from mlir_edsl import Tensor, f32, i32, rms_norm, token_logprobs
    from mlir_edsl.ast import Parameter
    P = lambda t: Parameter("p", t)
    x = P(Tensor[f32, 3, 8])
    for args, text in (((P(Tensor[f32, 8]),), "2D f32"), ((P(Tensor[i32, 3, 8]),), "2D f32"),
                       ((x, P(Tensor[f32, 7])), "columns"), ((x, P(Tensor[i32, 8])), "1D f32"),
                       ((x, None, P(Tensor[f32, 3, 7])), "residual")):
        with pytest.raises(TypeError, match=text):
            rms_norm(*args)
    with pytest.raises(ValueError, match="eps"):
        rms_norm(x, eps=0.0)
    for args, text in (((P(Tensor[i32, 3, 8]), P(Tensor[i32, 3])), "logits"),
                       ((x, P(Tensor[f32, 3])), "tokens"), ((x, P(Tensor[i32, 4])), "one token")):
        with pytest.raises(TypeError, match=text):
            token_logprobs(*args)


def test_register_weights_with_4_bits_refusals():
    import numpy as np
    from mlir_edsl import register_weights, release_weights
    W = np.ones((64, 8), np.float32)
    with pytest.raises(ValueError, match="4 or 32"):
        register_weights(W, bits=8)
    with pytest.raises(ValueError, match="group"):
        register_weights(W, bits=4, group=48)
    with pytest.raises(ValueError, match="not registered"):
        release_weights(W)
    register_weights(W, bits=4, group=32)  # nothing is packed before its first use
    register_weights(W, bits=4, group=64)
    release_weights(W)
    L = _native.lib()
    at = ctypes.c_void_p(W.ctypes.data)
    assert L.b200_weights_release_w4(at) == INVALID
    assert L.b200_weights_register_w4(at, 8, 64, 8, 33, 0) == INVALID
    assert L.b200_weights_register_w4(at, 7, 64, 8, 32, 0) == INVALID
    out = ctypes.c_void_p()
    assert L.b200_weights_w4(at, ctypes.byref(out)) == INVALID and not out.value
