"""The serving operators on the GPU against plain 64-bit formulas: norm with
residual and 8-bit output, 4-bit dense layer, token log probabilities.

Tolerances count roundings. A rounding to a type is off by at most half a
step: eps / 2 of the value (2^-24 f32, 2^-11 f16, 2^-8 bf16, 2^-4 e4m3), or
half the smallest step near zero."""
import math

import pytest
import torch

from mlir_edsl import _native, serving

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
HALF_TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25, E4M3: 2.0 ** -10}
INF, NAN = math.inf, math.nan


def half_step(v, dtype):
    """Half a step of `dtype` at the values v (float64)."""
    return (v.abs() * (torch.finfo(dtype).eps / 2)).clamp(min=HALF_TINY[dtype])


def rand(cuda, seed, *shape):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randn(*shape, device=cuda, generator=g)


def placed(t, pitch_more, offset):
    """t's values in a buffer with a wider pitch, `offset` elements into it."""
    m, n = t.shape
    buf = torch.zeros(offset + m * (n + pitch_more) + 64, dtype=torch.float32,
                      device=t.device).to(t.dtype)
    v = torch.as_strided(buf, (m, n), (n + pitch_more, 1), offset)
    v.copy_(t)
    return v


def synced():
    torch.cuda.synchronize()
    _native.check(_native.lib().b200_stream_sync(None))


# ------------------------------------------------------------------- rms_norm

# f32 work on a row: h, at most 32 squares in a thread, a tree of 10 + 5, the
# division, the square root and two products. Relative to y: half the sum's
# (32 + 15 + 2) roundings, and 6 more: below 32 * 2^-24.
NORM_F32 = 2.0 ** -19


def norm_formula(x, w, r, eps):
    h = x.double() + (r.double() if r is not None else 0)
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return y * w.double() if w is not None else y


def check_codes(codes, scales, y, group):
    m, n = y.shape
    group = group or n
    for i, g0 in enumerate(range(0, n, group)):
        part = y[:, g0:g0 + group]
        s = scales[:, i].double()
        most = part.abs().amax(1)
        want = torch.where(most > 0, most / 448, torch.ones_like(most))
        assert ((s - want).abs() <= 2 * NORM_F32 * want + 2.0 ** -149).all()
        value = codes[:, g0:g0 + group].double() * s[:, None]
        step = torch.maximum(half_step(part, E4M3), s[:, None] * HALF_TINY[E4M3])
        assert ((value - part).abs() <= step * (1 + 2.0 ** -10) + 4 * NORM_F32 * part.abs()).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,N", [(1, 1), (3, 7), (1, 4096), (130, 256), (33, 1001), (9, 2049),
                                 (5, 8192), (2, 16384), (3, 33000), (2, 100003)])
@pytest.mark.parametrize("residual,quant,group", [(False, None, 0), (True, None, 0),
                                                  (True, "e4m3", 0), (False, "e4m3", 32),
                                                  (True, "e4m3", 64), (True, "e4m3", 128)])
def test_rms_norm(cuda, dtype, M, N, residual, quant, group):
    x = (rand(cuda, N, M, N) * 2).to(dtype)
    r = (rand(cuda, N + 1, M, N) * 3).to(dtype) if residual else None
    w = (rand(cuda, N + 2, N) * 0.3 + 1).to(dtype)
    out = serving.rms_norm(x, w, residual=r, eps=1e-5, quant=quant, group=group)
    out = list(out) if isinstance(out, tuple) else [out]
    synced()
    if residual:
        h = out.pop()
        assert torch.equal(h, (x.float() + r.float()).to(dtype))
    y = norm_formula(x, w, r, 1e-5)
    if quant:
        assert out[0].dtype == E4M3 and out[1].shape == (M, -(-N // group) if group else 1)
        check_codes(out[0], out[1], y, group)
    else:
        assert out[0].dtype == dtype
        assert ((out[0].double() - y).abs() <= half_step(y, dtype) + NORM_F32 * y.abs()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [2, 149, 1190])
@pytest.mark.parametrize("chunks", [32, 33, 130, 257, 385, 513, 769, 1025, 1537, 2049, 2500])
@pytest.mark.parametrize("odd", [0, 1])
def test_rms_norm_widths(cuda, dtype, M, chunks, odd):
    """Rows of every number of 16-byte chunks where the threads of a row change,
    few of them, as many as run at once and more; on 16 bytes and cut off it."""
    if M * chunks > 1190 * 800:
        M = 301  # more than the CTAs that a GPU runs of the widest rows
    N = chunks * (4 if dtype == F32 else 8) - odd
    x = (rand(cuda, N, M, N) * 2).to(dtype)
    r = (rand(cuda, N + 1, M, N) * 3).to(dtype)
    w = (rand(cuda, N + 2, N) * 0.3 + 1).to(dtype)
    y, h = serving.rms_norm(x, w, residual=r, eps=1e-5)
    rows, row_scales, h1 = serving.rms_norm(x, w, residual=r, eps=1e-5, quant="e4m3")
    codes, scales, h2 = serving.rms_norm(x, w, residual=r, eps=1e-5, quant="e4m3", group=32)
    synced()
    for got in (h, h1, h2):
        assert torch.equal(got, (x.float() + r.float()).to(dtype))
    want = norm_formula(x, w, r, 1e-5)
    assert ((y.double() - want).abs() <= half_step(want, dtype) + NORM_F32 * want.abs()).all()
    check_codes(rows, row_scales, want, 0)
    some = slice(0, M, max(1, M // 7))
    check_codes(codes[some], scales[some], want[some], 32)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N,more,offset", [(512, 8, 0), (512, 3, 0), (512, 8, 1), (1000, 0, 5)])
def test_rms_norm_pitches_and_alignments(cuda, dtype, N, more, offset):
    x = placed(rand(cuda, 1, 11, N).to(dtype), more, offset)
    r = placed(rand(cuda, 2, 11, N).to(dtype), 0, 0)
    w = rand(cuda, 3, N)  # f32 weights with every type
    buf = torch.full((13, N + 5), 7.0, device=cuda).to(dtype)
    out = buf[1:12, :N]
    y, h = serving.rms_norm(x, w, residual=r, out=out)
    synced()
    want = norm_formula(x, w, r, 1e-6)
    assert y is out
    assert ((y.double() - want).abs() <= half_step(want, dtype) + NORM_F32 * want.abs()).all()
    assert (buf[0] == 7).all() and (buf[12] == 7).all() and (buf[:, N:] == 7).all()
    assert torch.equal(h, (x.float() + r.float()).to(dtype))


@pytest.mark.parametrize("N", [96, 4096, 40000])
@pytest.mark.parametrize("into", ["residual", "x"])
def test_rms_norm_residual_in_place(cuda, N, into):
    x, r = rand(cuda, 1, 37, N).bfloat16(), rand(cuda, 2, 37, N).bfloat16()
    want_y, want_h = serving.rms_norm(x, None, residual=r)
    a, b = x.clone(), r.clone()
    y, h = serving.rms_norm(a, None, residual=b, residual_out=a if into == "x" else b)
    synced()
    assert torch.equal(y, want_y) and torch.equal(h, want_h)
    assert torch.equal(a if into == "x" else b, want_h)


@pytest.mark.parametrize("N", [20001, 36000])
def test_rms_norm_long_rows_in_place_and_out_of_range(cuda, N):
    """Rows in shared memory: h over x, squares out of f32's range, zeros, a NaN."""
    x, r = rand(cuda, 1, 5, N), rand(cuda, 2, 5, N)
    x[1] *= 1e30
    x[2], r[2] = 0, 0
    x[3, N - 1] = NAN
    h = x + r
    want = norm_formula(x, None, r, 1e-6)
    y, got = serving.rms_norm(x, None, residual=r, residual_out=x)
    synced()
    assert got.data_ptr() == x.data_ptr()
    for row in (0, 1, 2, 4):
        assert torch.equal(x[row], h[row])
        err = (y[row].double() - want[row]).abs()
        # the sum: at most 18 partial sums of four in a thread, within the 32 above
        assert (err <= NORM_F32 * want[row].abs() + 2.0 ** -149).all(), row
    assert torch.isnan(y[3]).all()


def test_rms_norm_extreme_rows(cuda):
    """Squares out of f32's range, zeros, subnormal values, infinities, NaN."""
    N = 512
    x = rand(cuda, 1, 7, N)
    x[1] *= 1e30
    x[2] = 0
    x[3] = 1e-40
    x[4, 5] = INF
    x[5, 6] = NAN
    x[6] = 3e38
    y = serving.rms_norm(x, None)
    q, s = serving.rms_norm(x, None, quant="e4m3", group=64)
    synced()
    want = norm_formula(x, None, None, 1e-6)
    for row in (0, 1, 2, 3, 6):
        err = (y[row].double() - want[row]).abs()
        assert (err <= NORM_F32 * want[row].abs() + 2.0 ** -149).all(), row
    check_codes(q[[0, 1, 2, 6]], s[[0, 1, 2, 6]], want[[0, 1, 2, 6]], 64)
    assert (s[2] == 1).all() and (q[2].float() == 0).all()
    assert torch.isnan(y[4, 5]) and (y[4, :5] == 0).all()
    assert torch.isnan(y[5]).all() and torch.isnan(q[5].float()).all()


@pytest.mark.parametrize("w", [1e37, 1e-33, 1e-36, 0.0])
@pytest.mark.parametrize("N,group", [(512, 0), (512, 32), (301, 64), (301, 0)])
def test_rms_norm_codes_of_extreme_weights(cuda, w, N, group):
    x = rand(cuda, 1, 9, N)
    weight = torch.full((N,), w, device=cuda)
    q, s = serving.rms_norm(x, weight, quant="e4m3", group=group)
    synced()
    check_codes(q, s, norm_formula(x, weight, None, 1e-6), group)


def test_rms_norm_shapes(cuda):
    x = rand(cuda, 1, 2, 3, 64).half()
    y = serving.rms_norm(x, None)
    assert y.shape == x.shape
    assert torch.equal(y.reshape(6, 64), serving.rms_norm(x.reshape(6, 64), None))
    assert torch.equal(serving.rms_norm(x[0, 0], None), y[0, 0])
    assert serving.rms_norm(x[:0], None).shape == (0, 3, 64)
    q, s = serving.rms_norm(x, None, quant="e4m3", group=32)
    assert q.shape == x.shape and s.shape == (2, 3, 2)


# ------------------------------------------------------------------- dense_w4

def weights(cuda, seed, K, N, group, zeros, dtype):
    g = torch.Generator(device=cuda).manual_seed(seed)
    parts = -(-K // group)
    codes = torch.randint(0, 16, (K, N), device=cuda, generator=g, dtype=torch.uint8)
    scales = (torch.rand(parts, N, device=cuda, generator=g) + 0.5).to(dtype)
    z = (torch.randint(0, 16, (parts, N), device=cuda, generator=g, dtype=torch.uint8)
         if zeros else None)
    of = torch.arange(K, device=cuda) // group
    W = (codes.double() - (z.double()[of] if zeros else 8)) * scales.double()[of]
    return serving.pack_w4(codes, scales, z, group=group), W


def check_w4(y, x, W, bias, act, group, alpha=0.0, scale=None):
    """Sums in f32: within 64 of K at most four tensor-core steps of two
    truncations each (2^-22 of the sum of absolute products), then one addition
    for each group or 64 of K and 16 for the parts and warps and CTAs."""
    xd = x.double() if scale is None else x.double() * scale
    want, size = xd @ W, xd.abs() @ W.abs()
    K = W.shape[0]
    adds = -(-K // min(group, 32)) + 16
    bound = size * (2.0 ** -19 + adds * 2.0 ** -24)
    if scale is not None:
        bound += want.abs() * 2.0 ** -23
    if bias is not None:
        want = want + bias.double()
        bound += 2.0 ** -24 * want.abs()
    if act:
        want = torch.where(want > 0, want, alpha * want)
    bound += half_step(want, y.dtype)
    err = (y.double() - want).abs()
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("dtype", [F32, BF16, F16, E4M3])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (192, False)])
@pytest.mark.parametrize("M,K,N", [(1, 64, 64), (1, 1, 1), (2, 96, 17), (3, 4096, 512),
                                   (8, 1001, 999), (9, 640, 200), (17, 257, 130), (33, 2048, 65),
                                   (64, 511, 300), (65, 128, 129), (200, 320, 64)])
def test_dense_w4(cuda, dtype, group, zeros, M, K, N):
    held = BF16 if dtype == E4M3 else dtype
    w, W = weights(cuda, K + N, K, N, group, zeros, held)
    x = rand(cuda, M, M, K).to(dtype)
    bias = rand(cuda, 5, N).to(held) if zeros else None
    y = serving.dense_w4(x, w, bias, act=1 if zeros else 0)
    synced()
    assert y.dtype == held and y.shape == (M, N)
    check_w4(y, x, W, bias, 1 if zeros else 0, group)


@pytest.mark.parametrize("M,K,N", [(1, 16384, 128), (4, 11008, 320), (30, 8192, 1030)])
def test_dense_w4_long(cuda, M, K, N):
    for dtype in (F32, BF16):
        w, W = weights(cuda, 3, K, N, 128, True, dtype)
        x = rand(cuda, M, M, K).to(dtype)
        y = serving.dense_w4(x, w, act=2, alpha=0.25, out_dtype=F32)
        synced()
        check_w4(y, x, W, None, 2, 128, alpha=0.25)


@pytest.mark.parametrize("x_group", [0, 32, 64, 128])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", [(1, 96, 64), (5, 1000, 128), (40, 1024, 192)])
def test_dense_w4_scaled_rows(cuda, x_group, group, M, K, N):
    w, W = weights(cuda, 7, K, N, group, False, F16)
    x = rand(cuda, M, M, K).to(E4M3)
    parts = -(-K // x_group) if x_group else 1
    s = rand(cuda, 9, M, parts).abs() + 0.1
    y = serving.dense_w4(x, w, x_scales=s, x_group=x_group, out_dtype=F32)
    synced()
    per = s.double().repeat_interleave(x_group or K, 1)[:, :K]
    check_w4(y, x, W, None, 0, 32, scale=per)


def test_dense_w4_pitches_and_rows_behind(cuda):
    w, W = weights(cuda, 1, 320, 100, 64, True, F32)
    for dtype in (F32, BF16, F16, E4M3):
        for more, offset in ((0, 0), (8, 0), (3, 0), (16, 1)):
            x = placed(rand(cuda, 2, 6, 320).to(dtype), more, offset)
            buf = torch.full((8, 109), 7.0, device=cuda)
            y = serving.dense_w4(x, w, out=buf[1:7, :100])
            synced()
            check_w4(y, x, W, None, 0, 64)
            assert (buf[0] == 7).all() and (buf[7] == 7).all() and (buf[:, 100:] == 7).all()


def test_dense_w4_keeps_all_bits_of_f32(cuda):
    """One product in each row: x has 24 bits, the weight is a whole number."""
    K = 256
    codes = torch.full((K, 64), 8, dtype=torch.uint8, device=cuda)
    codes[3], codes[200] = 9, 15
    w = serving.pack_w4(codes, torch.ones(2, 64, device=cuda))
    x = torch.zeros(4, K, device=cuda)
    x[0, 3], x[1, 3], x[2, 200], x[3, 200] = 1 + 2.0 ** -23, -3.4e38, 1.7654321, 2.0 ** -100
    y = serving.dense_w4(x, w)
    synced()
    want = torch.stack([x[0, 3], x[1, 3], 7 * x[2, 200], 7 * x[3, 200]])
    assert torch.equal(y, want[:, None].expand(4, 64))


def test_dense_w4_not_finite_and_empty(cuda):
    w, W = weights(cuda, 1, 128, 64, 128, False, F32)
    x = rand(cuda, 1, 3, 128)
    x[0, 5], x[1, 6] = INF, NAN
    y = serving.dense_w4(x, w)
    synced()
    want = x.double() @ W
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(torch.isinf(y), torch.isinf(want))
    assert torch.equal(y[0][torch.isinf(y[0])], want[0][torch.isinf(want[0])].float())
    assert serving.dense_w4(x[:0], w).shape == (0, 64)
    none = serving.pack_w4(torch.empty(0, 64, dtype=torch.uint8, device=cuda),
                           torch.empty(0, 64, device=cuda))
    bias = rand(cuda, 2, 64)
    y = serving.dense_w4(torch.empty(3, 0, device=cuda), none, bias, act=1)
    assert torch.equal(y, bias.clamp(min=0).expand(3, 64))


@pytest.mark.parametrize("scale_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("K,N,group", [(256, 128, 128), (1001, 99, 32), (130, 70, 64)])
def test_quantize_and_dequantize(cuda, scale_dtype, K, N, group):
    W = rand(cuda, K, K, N)
    W[:, 3] = 0
    W[0, 4] = 1e-30
    w = serving.quantize_w4(W, group=group, scale_dtype=scale_dtype)
    got = w.dequantize()
    synced()
    assert w.shape == (K, N) and got.shape == (K, N)
    for k0 in range(0, K, group):
        part, back = W[k0:k0 + group].double(), got[k0:k0 + group].double()
        scale = part.abs().amax(0) / 7
        # half a step of the scale's grid; the scale's own rounding moves codes
        # of up to 8 scales
        room = scale * (0.5 + 8 * torch.finfo(scale_dtype).eps) + 1e-30
        assert ((part - back).abs() <= room).all()
    assert (got[:, 3] == 0).all()


def test_pack_and_dequantize_are_exact(cuda):
    for K, N, group, zeros in ((64, 64, 64, False), (200, 77, 32, True), (513, 130, 256, True)):
        w, W = weights(cuda, 5, K, N, group, zeros, F16)
        assert torch.equal(w.dequantize().double(), W)


# ------------------------------------------------------------- token_logprobs

def check_tokens(out, logits, tokens, top):
    # relative to the maximum: a sum's logarithm of a few units is lost next to
    # logits of a type's lowest value, even in 64 bits
    x = logits.double()
    x = x - x.amax(1, keepdim=True)
    T, V = x.shape
    lse = torch.logsumexp(x, 1)
    p = torch.softmax(x, 1)
    entropy = -torch.special.xlogy(p, p).sum(1)
    # e^t to 2 + 1.2 |t| steps of 2^-23, |t| e^t <= 0.37; sums of at most
    # V / 256 terms in a thread, half a step each (V / 512 steps), and 16 joins;
    # each join rescales (4 steps)
    s_err = (V / 512 + 4 + 16 * 5 + 8) * 2.0 ** -23
    span = (x.amax(1) - lse).abs() + 1
    if tokens is not None:
        given = tokens.long()
        at = x.gather(1, given.clamp(min=0)[:, None])[:, 0] - lse
        want = torch.where(given < 0, torch.zeros_like(at), at)
        fin = torch.isfinite(want)
        assert torch.equal(out.logprobs.double()[~fin], want[~fin])
        room = s_err + 2.0 ** -23 * (want.abs() + span)
        assert ((out.logprobs.double() - want).abs()[fin] <= room[fin]).all()
    else:
        assert out.logprobs is None
    assert ((out.entropy.double() - entropy).abs() <= (s_err + 2.0 ** -22) * (2 + 2 * entropy)).all()
    if top:
        order = torch.sort(x, dim=1, descending=True, stable=True)
        assert torch.equal(out.top_tokens.long(), order.indices[:, :top])
        want = order.values[:, :top] - lse[:, None]
        fin = torch.isfinite(want)
        assert torch.equal(torch.isinf(out.top_logprobs), ~fin)
        room = s_err + 2.0 ** -23 * (want.abs() + span[:, None])
        assert ((out.top_logprobs.double() - want).abs()[fin] <= room[fin]).all()
    else:
        assert out.top_logprobs is None and out.top_tokens is None


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,V", [(1, 1), (2, 5), (1, 131072), (3, 32001), (700, 1000), (5, 4097),
                                 (17, 50257), (2, 200003)])
@pytest.mark.parametrize("top", [0, 1, 20, 32])
def test_token_logprobs(cuda, dtype, T, V, top):
    top = min(top, V)
    logits = (rand(cuda, V, T, V) * 3).to(dtype)
    tokens = torch.arange(T, device=cuda, dtype=torch.int32) * 977 % V
    tokens[T // 2] = -1 if T > 1 else V - 1
    out = serving.token_logprobs(logits, tokens, top=top)
    synced()
    check_tokens(out, logits, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [300, 40000])
def test_token_logprobs_of_ties(cuda, dtype, V):
    """Few different values: the lowest index comes first."""
    logits = torch.zeros(6, V, device=cuda)
    logits[1] = torch.arange(V, device=cuda) % 3
    logits[2] = -(torch.arange(V, device=cuda) % 2).float() * 0.0  # 0 and -0 are equal
    logits[3] = torch.arange(V, device=cuda).float() / V           # ascending
    logits[4, V // 2:] = 5
    logits[5, -3:] = 1
    logits = logits.to(dtype)
    out = serving.token_logprobs(logits, top=32)
    synced()
    check_tokens(out, logits, None, 32)


def test_token_logprobs_of_one_thread(cuda):
    """The most probable tokens all in the chunks that one thread reads."""
    V = 512 * 8 * 40
    logits = rand(cuda, 1, 2, V).bfloat16()
    at = torch.arange(40, device=cuda) * 512 * 8
    logits[:, at] = (20 + torch.arange(40, device=cuda).float()).bfloat16()
    logits[:, at + 1] = 21
    out = serving.token_logprobs(logits, top=32)
    synced()
    check_tokens(out, logits, None, 32)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [100, 30011])
def test_token_logprobs_of_masked_rows(cuda, dtype, V):
    logits = rand(cuda, 1, 5, V).to(dtype)
    low = torch.finfo(dtype).min
    logits[0, 3:] = -INF            # fewer tokens than alternatives
    logits[1, ::2] = -INF
    logits[2] = low                 # the type's lowest value everywhere
    logits[3, 1:] = low
    logits[4, : V // 2] = low
    logits[4, V // 2:] = -INF
    tokens = torch.tensor([50, 1, 2, 0, V // 2], dtype=torch.int32, device=cuda)
    out = serving.token_logprobs(logits, tokens, top=10)
    synced()
    check_tokens(out, logits, tokens, 10)


def test_token_logprobs_of_rows_without_a_distribution(cuda):
    for V in (64, 70000):
        logits = rand(cuda, 1, 4, V)
        logits[0] = -INF
        logits[1, 7], logits[2, V - 1] = NAN, INF
        tokens = torch.tensor([0, 1, 2, V], dtype=torch.int32, device=cuda)
        out = serving.token_logprobs(logits, tokens, top=4)
        synced()
        assert out.logprobs[0] == -INF and out.entropy[0] == 0
        assert (out.top_logprobs[0] == -INF).all()
        assert out.top_tokens[0].tolist() == [0, 1, 2, 3]
        assert torch.isnan(out.logprobs[1:]).all()  # the last: a token past V
        assert torch.isnan(out.entropy[1:3]).all() and torch.isfinite(out.entropy[3])
        assert torch.isnan(out.top_logprobs[1:3]).all()
        order = torch.sort(torch.nan_to_num(logits, nan=-INF, posinf=INF, neginf=-INF), dim=1,
                           descending=True, stable=True).indices
        assert torch.equal(out.top_tokens.long(), order[:, :4])


@pytest.mark.parametrize("more,offset", [(0, 1), (5, 0), (8, 3)])
def test_token_logprobs_pitches(cuda, more, offset):
    for dtype in (F32, F16):
        logits = placed((rand(cuda, 1, 9, 5000) * 2).to(dtype), more, offset)
        tokens = torch.arange(9, dtype=torch.int32, device=cuda)
        out = serving.token_logprobs(logits, tokens, top=3)
        synced()
        check_tokens(out, logits, tokens, 3)
    cube = (rand(cuda, 2, 2, 3, 100) * 2).half()
    out = serving.token_logprobs(cube, torch.zeros(2, 3, dtype=torch.int32, device=cuda), top=2)
    assert out.logprobs.shape == (2, 3) and out.top_tokens.shape == (2, 3, 2)
    assert serving.token_logprobs(cube[:0]).entropy.shape == (0, 3)


# ------------------------------------------------------------------- together

def network(cuda, seed=0, width=512, inner=1408, vocabulary=2003):
    torch.manual_seed(seed)
    W = [torch.randn(width, inner, device=cuda) / width ** 0.5,
         torch.randn(inner, width, device=cuda) / inner ** 0.5,
         torch.randn(width, vocabulary, device=cuda) / width ** 0.5]
    packed = [serving.quantize_w4(w, group=g, scale_dtype=BF16) for w, g in zip(W, (128, 64, 32))]
    norms = [torch.rand(width, device=cuda) + 0.5 for _ in range(2)]
    return packed, norms


def step(packed, norms, h, delta, tokens):
    """One layer and the head of a network of dense layers, as it is served."""
    q, s, h = serving.rms_norm(delta, norms[0], residual=h, quant="e4m3", group=128)
    a = serving.dense_w4(q, packed[0], act=1, x_scales=s, x_group=128)
    delta = serving.dense_w4(a, packed[1])
    q, s, h = serving.rms_norm(delta, norms[1], residual=h, quant="e4m3")
    logits = serving.dense_w4(q, packed[2], x_scales=s, out_dtype=F32)
    return h, logits, serving.token_logprobs(logits, tokens, top=5)


def test_a_served_step(cuda):
    """The operators in a row against the formulas, each on the outputs of the
    one before, and the same step again, on another stream and in a graph."""
    packed, norms = network(cuda)
    h0, d0 = rand(cuda, 1, 6, 512).bfloat16(), rand(cuda, 2, 6, 512).bfloat16()
    tokens = torch.tensor([1, 5, 2002, -1, 7, 8], dtype=torch.int32, device=cuda)
    q, s, h1 = serving.rms_norm(d0, norms[0], residual=h0, quant="e4m3", group=128)
    y = norm_formula(d0, norms[0], h0, 1e-6)
    check_codes(q, s, y, 128)
    a = serving.dense_w4(q, packed[0], act=1, x_scales=s, x_group=128)
    check_w4(a, q, packed[0].dequantize().double(), None, 1, 32,
             scale=s.double().repeat_interleave(128, 1))
    d1 = serving.dense_w4(a, packed[1])
    check_w4(d1, a, packed[1].dequantize().double(), None, 0, 64)
    h, logits, scores = step(packed, norms, h0, d0, tokens)
    synced()
    assert torch.equal(h, (d1.float() + h1.float()).bfloat16())
    check_tokens(scores, logits, tokens, 5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(packed, norms, h0, d0, tokens)
    torch.cuda.current_stream().wait_stream(side)
    synced()
    assert torch.equal(other[1], logits) and torch.equal(other[2].top_tokens, scores.top_tokens)

    graphs = []
    for _ in range(2):  # two graphs that run side by side share nothing
        hs, ds = h0.clone(), d0.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(packed, norms, hs, ds, tokens)
        graphs.append((g, hs, ds, out))
    new = [(rand(cuda, 10 + i, 6, 512).bfloat16(), rand(cuda, 20 + i, 6, 512).bfloat16())
           for i in range(2)]
    for _ in range(3):
        streams = [torch.cuda.Stream() for _ in graphs]
        for (g, hs, ds, _), (a, b), st in zip(graphs, new, streams):
            hs.copy_(a)
            ds.copy_(b)
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        synced()
        for (_, _, _, out), (a, b) in zip(graphs, new):
            want = step(packed, norms, a, b, tokens)
            synced()
            assert torch.equal(out[1], want[1])
            assert torch.equal(out[2].logprobs, want[2].logprobs)


def test_results_do_not_change_between_calls(cuda):
    packed, norms = network(cuda, seed=3, vocabulary=50001)
    h, d = rand(cuda, 1, 2, 512).bfloat16(), rand(cuda, 2, 2, 512).bfloat16()
    tokens = torch.tensor([4, 5], dtype=torch.int32, device=cuda)
    first = step(packed, norms, h, d, tokens)
    for _ in range(20):
        again = step(packed, norms, h, d, tokens)
        for a, b in zip((first[0], first[1], *first[2]), (again[0], again[1], *again[2])):
            assert torch.equal(a, b)


def test_gradients_are_refused(cuda):
    x = rand(cuda, 1, 2, 64).requires_grad_()
    with pytest.raises(ValueError, match="no backward pass"):
        serving.rms_norm(x)
    with torch.no_grad():
        serving.rms_norm(x)
    with pytest.raises(ValueError, match="no backward pass"):
        serving.token_logprobs(x)


# ------------------------------------------------------------------- frontend

@pytest.mark.parametrize("M", [1, 7, 300])
@pytest.mark.parametrize("bits,group", [(32, 128), (4, 32), (4, 128)])
def test_frontend_network(cuda, M, bits, group):
    """norm -> dense layer -> dense layer -> log probabilities as one traced
    function, with f32 weights and with weights registered in 4 bits. Errors
    are carried through: of the norm, then of each layer 2^-18 of the sum of
    absolute products (3xTF32 drops 2^-20 of it, the 4-bit layer 2^-19), then
    twice the row's largest."""
    import numpy as np
    from mlir_edsl import (Tensor, f32, get_backend, i32, ml_function, register_weights,
                           release_weights, relu, rms_norm, token_logprobs)
    K, H, V = 200, 320, 517
    rng = np.random.default_rng(M)
    X, R = (rng.standard_normal((M, K)).astype(np.float32) for _ in range(2))
    w = (1 + 0.1 * rng.standard_normal(K)).astype(np.float32)
    W1 = (rng.standard_normal((K, H)) / K ** 0.5).astype(np.float32)
    b1 = rng.standard_normal(H).astype(np.float32)
    W2 = (rng.standard_normal((H, V)) / H ** 0.5).astype(np.float32)
    tokens = rng.integers(0, V, M).astype(np.int32)
    tokens[-1] = -1 if M > 1 else tokens[-1]

    @ml_function(target="b200")
    def net(X: Tensor[f32, M, K], R: Tensor[f32, M, K], w: Tensor[f32, K], W1: Tensor[f32, K, H],
            b1: Tensor[f32, H], W2: Tensor[f32, H, V], tokens: Tensor[i32, M]) -> Tensor[f32, M]:
        return token_logprobs(relu(rms_norm(X, w, R) @ W1 + b1) @ W2, tokens)

    D1, D2 = torch.from_numpy(W1).to(cuda), torch.from_numpy(W2).to(cuda)
    if bits == 4:
        D1, D2 = (serving.quantize_w4(d, group=group).dequantize() for d in (D1, D2))
        register_weights(W1, bits=4, group=group)
        register_weights(W2, bits=4, group=group)
    try:
        got = net(X, R, w, W1, b1, W2, tokens)
        again = net(X, R, w, W1, b1, W2, tokens)
        if bits == 4 and M <= 256:
            assert get_backend().last_launches == 4  # one kernel a step, nothing packed again
    finally:
        if bits == 4:
            release_weights(W1)
            release_weights(W2)
    assert got.shape == (M,) and np.array_equal(got, again)
    D1, D2 = D1.double(), D2.double()
    x, r, bd = (torch.from_numpy(a).to(cuda) for a in (X, R, b1))
    y = norm_formula(x, torch.from_numpy(w).to(cuda), r, 1e-6)
    err = NORM_F32 * y.abs()
    a = y @ D1 + bd.double()
    err = err @ D1.abs() + 2.0 ** -18 * (y.abs() @ D1.abs()) + 2.0 ** -23 * a.abs()
    a = a.clamp(min=0)
    logits = a @ D2
    err = err @ D2.abs() + 2.0 ** -18 * (a.abs() @ D2.abs())
    t = torch.from_numpy(tokens).to(cuda).long()
    want = torch.log_softmax(logits, 1).gather(1, t.clamp(min=0)[:, None])[:, 0]
    want = torch.where(t < 0, torch.zeros_like(want), want)
    room = 2 * err.amax(1) + 2.0 ** -16
    diff = (torch.from_numpy(got).to(cuda).double() - want).abs()
    assert (diff <= room).all(), (diff / room).max()


def test_frontend_4_bit_weights_follow_versions(cuda):
    import numpy as np
    from mlir_edsl import Tensor, f32, ml_function, register_weights, release_weights
    W = np.ones((64, 64), np.float32)
    X = np.ones((2, 64), np.float32)

    @ml_function(target="b200")
    def f(X: Tensor[f32, 2, 64], W: Tensor[f32, 64, 64]) -> Tensor[f32, 2, 64]:
        return X @ W

    register_weights(W, 1, bits=4, group=64)
    try:
        np.testing.assert_allclose(f(X, W), 64, rtol=2.0 ** -20)
        W *= 2
        np.testing.assert_allclose(f(X, W), 64, rtol=2.0 ** -20)  # the documented contract
        register_weights(W, 2, bits=4, group=64)
        np.testing.assert_allclose(f(X, W), 128, rtol=2.0 ** -20)
        _native.check(_native.lib().b200_release())  # copies are made again
        np.testing.assert_allclose(f(X, W), 128, rtol=2.0 ** -20)
        register_weights(W, 2)  # back to 32 bits
        np.testing.assert_array_equal(f(X, W), 128)
    finally:
        release_weights(W)
    np.testing.assert_array_equal(f(X, W), 128)
