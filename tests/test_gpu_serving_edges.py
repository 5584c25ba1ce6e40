"""The serving operators at the edges of what they take: the longest rows, values
at both ends of f32's range, buffers that overlap, waits that run out."""
import math

import pytest
import torch

from mlir_edsl import _native, serving

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
INF, NAN = math.inf, math.nan


def rand(cuda, seed, *shape):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randn(*shape, device=cuda, generator=g)


def synced():
    torch.cuda.synchronize()
    _native.check(_native.lib().b200_stream_sync(None))


def test_dense_w4_rows_past_2_to_30(cuda):
    """A row's bytes pass 2^31: every element counts, the first and last blocks'
    among them. Whole numbers, so the sums are exact."""
    K = (1 << 30) + 320
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 72 << 30:
        pytest.skip("needs 72 GB of device memory")
    x = torch.zeros(9, K, dtype=BF16, device=cuda)
    at = [0, 70, 319, 320, K // 2, K - 321, K - 1]
    for i, k in enumerate(at):
        x[:, k] = 1 << i
    x[3, at[1]] = 0
    codes = torch.full((K, 1), 9, dtype=torch.uint8, device=cuda)
    w = serving.pack_w4(codes, torch.ones(2, 1, dtype=BF16, device=cuda), group=1 << 30)
    del codes
    try:
        y = serving.dense_w4(x, w, out_dtype=F32)
        synced()
        want = torch.full((9, 1), 127.0, device=cuda)
        want[3] -= 2
        assert torch.equal(y, want)
    finally:
        del x, w
        torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [1, 2, 3, 9, 70])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_dense_w4_sums_past_the_range(cuda, dtype, M, group):
    """Sums of x * (code - zero) that leave f32's range while those of x * W stay in
    it. Terms of one sign: a sum of absolute products is the sum itself, so its
    error is below 2^-18 of it (16 k16 steps of two truncations, 2^-22 each, no more
    than 8 of them in one sum; 8 + 16 additions)."""
    K, N = 256, 70
    codes = torch.full((K, N), 15, dtype=torch.uint8, device=cuda)
    zeros = torch.zeros(-(-K // group), N, dtype=torch.uint8, device=cuda)
    scales = torch.full(zeros.shape, 2.0 ** -16, device=cuda)
    w = serving.pack_w4(codes, scales, zeros, group=group)
    for value in (3e38, -1e38, 1e30):
        x = torch.full((M, K), value, device=cuda).to(dtype)
        y = serving.dense_w4(x, w, out_dtype=F32)
        synced()
        want = x.double().sum(1, keepdim=True) * (15 * 2.0 ** -16)
        assert ((y.double() - want).abs() <= 2.0 ** -18 * want.abs()).all()


# as in the tests of ordinary rows: 49 roundings of the sum, halved by the root,
# and six more; one of these is that of a row's second factor
NORM_F32 = 2.0 ** -19


def norm_formula(x, eps):
    h = x.double()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)


def half_step(v, dtype):
    tiny = {F32: 2.0 ** -150, BF16: 2.0 ** -134}[dtype]
    return (v.abs() * (torch.finfo(dtype).eps / 2)).clamp(min=tiny)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [301, 512, 4096, 20001, 50000])
def test_rms_norm_of_small_values_beside_large_ones(cuda, dtype, N):
    """A row whose squares leave f32's range keeps the bits of its small values."""
    x = rand(cuda, N, 5, N) * 1e-12
    x[0, 0], x[1, N - 1], x[2, 7], x[3, 9] = 2e19, -3e38, 1e25, 5e19
    x[4, ::3] = 1e22
    x = x.to(dtype)
    y = serving.rms_norm(x)
    q, s = serving.rms_norm(x, quant="e4m3", group=32)
    synced()
    want = norm_formula(x, 1e-6)
    assert ((y.double() - want).abs() <= half_step(want, dtype) + NORM_F32 * want.abs()).all()
    for i, g0 in enumerate(range(0, N, 32)):
        most = want[:, g0:g0 + 32].abs().amax(1)
        scale = s[:, i].double()
        # a scale below half of f32's smallest value is 0 there, and 1 stands for 0
        none = (most / 448 < 2.0 ** -149) & (scale == 1)
        room = 2 * NORM_F32 * most / 448 + 2.0 ** -149
        assert (none | ((scale - most / 448).abs() <= room)).all()


@pytest.mark.parametrize("N", [301, 512, 4096, 20001, 50000])
def test_rms_norm_of_tiny_rows_and_eps(cuda, N):
    """Squares below f32's range, with an eps that does not hide them."""
    eps = float(torch.tensor(1e-42))
    x = rand(cuda, N, 4, N) * 1e-21
    x[1] *= 1e-3
    x[2] = 0
    x[3] *= 1e5
    y = serving.rms_norm(x, eps=eps)
    synced()
    want = norm_formula(x, eps)
    assert ((y.double() - want).abs() <= half_step(want, F32) + NORM_F32 * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16, E4M3])
@pytest.mark.parametrize("M,K,group", [(9, 64, 64), (40, 4096, 128), (100, 1000, 32)])
def test_dense_w4_waits_that_run_out(cuda, dtype, M, K, group):
    """Waits for products that never report their end give up after 1 ms: the
    result is NaN throughout, check() raises once, the next call is right."""
    w = serving.quantize_w4(rand(cuda, 1, K, 300), group=group)
    x = rand(cuda, 2, M, K).to(dtype)
    want = serving.dense_w4(x, w, act=1, out_dtype=BF16)
    serving.check()
    expire = _native.lib().b200_debug_w4_expire
    _native.check(expire(1_000_000))
    try:
        y = serving.dense_w4(x, w, act=1, out_dtype=BF16)
        with pytest.raises(_native.B200Error, match="bounded wait") as e:
            serving.check()
    finally:
        _native.check(expire(0))
    assert e.value.code == 5 and torch.isnan(y).all()
    serving.check(cuda)
    assert torch.equal(serving.dense_w4(x, w, act=1, out_dtype=BF16), want)
    serving.check()


@pytest.mark.parametrize("scale_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_quantize_of_weights_that_are_not_finite(cuda, scale_dtype, value):
    """A weight that is no number shows: its group of its column is NaN, and
    nothing else changes."""
    W = rand(cuda, 1, 200, 40)
    clean = serving.quantize_w4(W, group=64, scale_dtype=scale_dtype).dequantize()
    W[70, 3] = value
    got = serving.quantize_w4(W, group=64, scale_dtype=scale_dtype).dequantize()
    synced()
    assert torch.isnan(got[64:128, 3]).all()
    got[64:128, 3] = clean[64:128, 3]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,N", [(1, 1), (5, 4096), (300, 1001), (40, 8200), (3, 20001), (2, 100003)])
def test_rms_norm_over_its_inputs(cuda, dtype, M, N):
    """The result may take the place of x or of the residual."""
    x, r = (rand(cuda, 1, M, N) * 2).to(dtype), rand(cuda, 2, M, N).to(dtype)
    want = serving.rms_norm(x)
    want_y, want_h = serving.rms_norm(x, residual=r)
    a = x.clone()
    assert serving.rms_norm(a, out=a) is a
    b, c = x.clone(), r.clone()
    serving.rms_norm(b, residual=c, out=b, residual_out=c)
    d, e = x.clone(), r.clone()
    _, h = serving.rms_norm(d, residual=e, out=e)
    synced()
    assert torch.equal(a, want)
    assert torch.equal(b, want_y) and torch.equal(c, want_h)
    assert torch.equal(e, want_y) and torch.equal(h, want_h)


def test_outputs_that_overlap_are_refused(cuda):
    buf = rand(cuda, 1, 8, 512)
    x, r = buf[1:5, :128], buf[1:5, 128:256]
    side = buf[1:5, 256:384]
    serving.rms_norm(x, residual=r, out=side)  # columns of one buffer, side by side
    weight = rand(cuda, 2, 1024)[:128]
    for kw in (dict(out=buf[2:6, :128]), dict(out=buf[1:5, 64:192]),
               dict(out=side, residual_out=side), dict(residual_out=buf[0:4, 128:256])):
        with pytest.raises(ValueError, match="overlap"):
            serving.rms_norm(x, residual=r, **kw)
    line = rand(cuda, 2, 128)
    with pytest.raises(ValueError, match="overlap"):
        serving.rms_norm(x[:1], line, out=line[None])
    with pytest.raises(ValueError, match="overlap"):
        serving.rms_norm(rand(cuda, 2, 1, 128), weight, quant="e4m3",
                         out=weight.view(torch.float8_e4m3fn)[None, :128])
    w = serving.quantize_w4(rand(cuda, 3, 128, 128), group=64)
    serving.dense_w4(x, w, out=side)
    bias = rand(cuda, 4, 4, 128)
    with pytest.raises(ValueError, match="overlap"):
        serving.dense_w4(x, w, out=x)
    with pytest.raises(ValueError, match="overlap"):
        serving.dense_w4(x, w, out=buf[3:7, 100:228])
    with pytest.raises(ValueError, match="overlap"):
        serving.dense_w4(x, w, bias[2], out=bias)
    with pytest.raises(ValueError, match="overlap"):
        serving.dense_w4(x[:1], w, out=w.buffer.view(F32)[None, :128])
    s = torch.ones(4, 128, device=cuda)
    with pytest.raises(ValueError, match="overlap"):
        serving.dense_w4(x.to(E4M3), w, x_scales=s[:, :2], x_group=64, out=s)
    synced()


def test_outputs_count_as_changed(cuda):
    """A tensor that a backward pass needs and that a call overwrites is noticed."""
    x, r = rand(cuda, 1, 4, 64), rand(cuda, 2, 4, 64)
    out, h = torch.ones_like(x), torch.ones_like(x)
    leaf = torch.ones(4, 64, device=cuda, requires_grad=True)
    loss = (leaf * out).sum()
    before = out._version, h._version, x._version
    serving.rms_norm(x, residual=r, out=out, residual_out=h)
    assert (out._version, h._version, x._version) == (before[0] + 1, before[1] + 1, before[2])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    w = serving.quantize_w4(rand(cuda, 3, 64, 64), group=64)
    serving.dense_w4(x, w, out=out)
    assert out._version == before[0] + 2
    serving.rms_norm(x, residual=r, residual_out=r)  # one change, not two
    assert r._version == 1
    with pytest.raises(ValueError):
        serving.dense_w4(x, w, out=h[:2])
    assert h._version == before[1] + 1  # a refused call changes nothing
    with torch.inference_mode():
        kept = torch.empty_like(x)
    serving.rms_norm(x, out=kept)  # has no version
    synced()


def test_forward_gradients_are_refused(cuda):
    import torch.autograd.forward_ad as forward
    x = rand(cuda, 1, 2, 64)
    w = serving.quantize_w4(rand(cuda, 2, 64, 64), group=64)
    with forward.dual_level():
        dual = forward.make_dual(x, torch.ones_like(x))
        for call in (lambda: serving.rms_norm(dual), lambda: serving.dense_w4(dual, w),
                     lambda: serving.token_logprobs(dual), lambda: serving.quantize_w4(dual),
                     lambda: serving.rms_norm(x, dual[0]),
                     lambda: serving.rms_norm(x, residual=dual)):
            with pytest.raises(ValueError, match="forward"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="forward"):
                call()
        serving.rms_norm(forward.unpack_dual(dual).primal)
    synced()


def test_negated_views_are_refused(cuda):
    """A view that stands for the negative of its memory (the imaginary part of a
    conjugate, for example)."""
    part = torch.complex(rand(cuda, 1, 3, 1), rand(cuda, 2, 3, 1)).conj().imag
    with pytest.raises(ValueError, match="resolve_neg"):
        serving.rms_norm(part)
    x = rand(cuda, 3, 3, 64)
    with pytest.raises(ValueError, match="resolve_neg"):
        serving.token_logprobs(torch._neg_view(x))
    with pytest.raises(ValueError, match="resolve_neg"):
        serving.rms_norm(x, out=torch._neg_view(x.clone()))
    serving.rms_norm(part.resolve_neg())
    synced()


def test_rms_norm_scales_of_rows_without_columns(cuda):
    junk = torch.full((64,), 7.0, device=cuda)
    del junk  # the allocator hands its memory to the scales
    x = torch.empty(5, 0, device=cuda)
    q, s = serving.rms_norm(x, quant="e4m3")
    synced()
    assert q.shape == (5, 0) and (s == 1).all() and s.shape == (5, 1)
    q, s = serving.rms_norm(x, torch.empty(0, device=cuda), quant="e4m3", group=32)
    synced()
    assert q.shape == (5, 0) and s.shape == (5, 0)


# ----------------------------------------------- forms of calls not tested elsewhere

@pytest.mark.parametrize("dtype", [F32, BF16, F16, E4M3])
@pytest.mark.parametrize("M", [3, 20, 100])
def test_dense_w4_without_columns_of_x(cuda, dtype, M):
    none = serving.pack_w4(torch.empty(0, 130, dtype=torch.uint8, device=cuda),
                           torch.empty(0, 130, device=cuda))
    bias = rand(cuda, 2, 130)
    y = serving.dense_w4(torch.empty(M, 0, device=cuda, dtype=dtype), none, bias, act=1,
                         out_dtype=F32)
    synced()
    assert torch.equal(y, bias.clamp(min=0).expand(M, 130))


@pytest.mark.parametrize("M", [1, 2, 4])
def test_dense_w4_keeps_all_bits_of_f32_rows(cuda, M):
    """One product in each row, on both kernels: up to 2 rows of f32 and more."""
    K = 256
    codes = torch.full((K, 64), 8, dtype=torch.uint8, device=cuda)
    codes[3], codes[200] = 9, 15
    w = serving.pack_w4(codes, torch.ones(2, 64, device=cuda))
    for at, value in ((3, 1 + 2.0 ** -23), (3, -3.4e38), (200, 1.7654321), (200, 2.0 ** -100),
                      (3, 1.9999999), (3, -1.0000001e-20)):
        x = torch.zeros(M, K, device=cuda)
        x[M - 1, at] = value
        y = serving.dense_w4(x, w)
        synced()
        want = (x[:, at].double() * (1 if at == 3 else 7)).float()
        assert torch.equal(y, want[:, None].expand(M, 64))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 2, 8, 9, 33, 100])
def test_dense_w4_sums_by_unit(cuda, dtype, group, M):
    """Errors against the additions that the kernels make: within a unit of K
    (32 in groups of 32; 128 in groups of 128 on the tensor core; otherwise 64)
    one k16 step after another, two truncations of 2^-22 of the sum of absolute
    products each; then one f32 addition a unit and 16 for parts, warps, CTAs."""
    K, N = 4096, 192
    g = torch.Generator(device=cuda).manual_seed(M)
    codes = torch.randint(0, 16, (K, N), device=cuda, generator=g, dtype=torch.uint8)
    scales = (torch.rand(K // group, N, device=cuda, generator=g) + 0.5).to(dtype)
    W = (codes.double() - 8) * scales.double()[torch.arange(K, device=cuda) // group]
    x = rand(cuda, M, M, K).to(dtype)
    y = serving.dense_w4(x, serving.pack_w4(codes, scales, group=group), out_dtype=F32)
    synced()
    columns = M * (3 if dtype == F32 else 1)
    unit = 32 if group == 32 else 128 if group == 128 and columns > 8 else 64
    room = unit / 16 * 2 * 2.0 ** -22 + (K // unit + 16) * 2.0 ** -24 + 2.0 ** -24
    size = x.double().abs() @ W.abs()
    assert ((y.double() - x.double() @ W).abs() <= room * size).all()


@pytest.mark.parametrize("x_group", [32, 64, 128])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_dense_w4_many_scaled_rows(cuda, x_group, group):
    M, K, N = 100, 1000, 192
    g = torch.Generator(device=cuda).manual_seed(7)
    codes = torch.randint(0, 16, (K, N), device=cuda, generator=g, dtype=torch.uint8)
    parts = -(-K // group)
    scales = torch.rand(parts, N, device=cuda, generator=g) + 0.5
    W = (codes.double() - 8) * scales.double()[torch.arange(K, device=cuda) // group]
    x = rand(cuda, M, M, K).to(E4M3)
    s = rand(cuda, 9, M, -(-K // x_group)).abs() + 0.1
    y = serving.dense_w4(x, serving.pack_w4(codes, scales, group=group), x_scales=s,
                         x_group=x_group, out_dtype=F32)
    synced()
    xd = x.double() * s.double().repeat_interleave(x_group, 1)[:, :K]
    size = xd.abs() @ W.abs()
    # as above with the smallest unit's additions and the longest unit's steps,
    # and one rounding more for the second scale
    room = 16 * 2.0 ** -22 + (K / 32 + 16 + 2) * 2.0 ** -24
    assert ((y.double() - xd @ W).abs() <= room * size).all()


def test_token_logprobs_of_many_rows_in_one_thread(cuda):
    """Rows of one CTA each whose most probable tokens all lie in the 16-byte
    chunks of one of its 256 threads."""
    T, V = 300, 256 * 8 * 40
    logits = rand(cuda, 1, T, V).bfloat16()
    at = torch.arange(40, device=cuda) * 256 * 8 + 24
    logits[:, at] = (20 + torch.arange(40, device=cuda).float()).bfloat16()
    logits[:, at + 1] = 21
    out = serving.token_logprobs(logits, top=32)
    synced()
    for i in range(0, T, 50):
        x = logits[i:i + 50].double()
        order = torch.sort(x, dim=1, descending=True, stable=True)
        assert torch.equal(out.top_tokens[i:i + 50].long(), order.indices[:, :32])
        want = order.values[:, :32] - torch.logsumexp(x, 1, keepdim=True)
        # e^t to some steps of 2^-23, at most 320 of them in a thread's sum, 16 joins
        room = (320 / 2 + 92) * 2.0 ** -23 + 2.0 ** -22 * (want.abs() + 64)
        assert ((out.top_logprobs[i:i + 50].double() - want).abs() <= room).all()


def test_calls_from_several_threads(cuda):
    """Threads on streams of their own get what one thread gets."""
    import threading
    w = serving.quantize_w4(rand(cuda, 1, 512, 3001), group=64)
    norm = rand(cuda, 2, 512)
    rows = [rand(cuda, 3 + i, 1 + 7 * i, 512).bfloat16() for i in range(4)]

    def served(x):
        q, s, h = serving.rms_norm(x, norm, residual=x, quant="e4m3", group=128)
        logits = serving.dense_w4(q, w, x_scales=s, x_group=128, out_dtype=F32)
        return (h, logits) + serving.token_logprobs(logits, top=7)[1:]

    want = [served(x) for x in rows]
    synced()
    got, wrong = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()) as _:
                for _ in range(50):
                    got[i] = served(rows[i])
                    if not all(torch.equal(a, b) for a, b in zip(got[i], want[i])):
                        wrong.append(i)
                with pytest.raises(ValueError):
                    serving.rms_norm(rows[i], group=i + 1)
        except BaseException as e:  # a thread's failure is the test's
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    synced()
    assert not wrong, wrong


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [2, 20])
def test_dense_w4_of_tiny_rows(cuda, dtype, M):
    """Sums are kept divided by 4096, so bits below 2^-149 * 4096 = 2^-137 are lost:
    no more than two such steps for each of K products, times the scale. And the
    bf16 parts of an f32 x have no bits below bf16's smallest value, 2^-133: less
    than that is lost of each x."""
    K, N = 128, 70
    g = torch.Generator(device=cuda).manual_seed(M)
    codes = torch.randint(0, 16, (K, N), device=cuda, generator=g, dtype=torch.uint8)
    scales = torch.rand(2, N, device=cuda, generator=g) + 0.5
    W = (codes.double() - 8) * scales.double()[torch.arange(K, device=cuda) // 64]
    x = (rand(cuda, M, M, K) * 2.0 ** -118).to(dtype)
    y = serving.dense_w4(x, serving.pack_w4(codes, scales, group=64), out_dtype=F32)
    synced()
    size = x.double().abs() @ W.abs()
    room = 2 * K * 1.5 * 2.0 ** -137 + 2.0 ** -18 * size
    if dtype == F32:
        room = room + 2.0 ** -133 * W.abs().sum(0)
    assert ((y.double() - x.double() @ W).abs() <= room).all()


def test_frontend_operators_alone_and_4_bits_on_the_left(cuda):
    """Functions of one step; weights in 4 bits count where they are the right
    operand of a product, and as f32 everywhere else."""
    import numpy as np
    from mlir_edsl import (Tensor, f32, i32, ml_function, register_weights, release_weights,
                           rms_norm, token_logprobs)

    @ml_function(target="b200")
    def norm(X: Tensor[f32, 5, 64]) -> Tensor[f32, 5, 64]:
        return rms_norm(X)

    @ml_function(target="b200")
    def score(X: Tensor[f32, 5, 64], t: Tensor[i32, 5]) -> Tensor[f32, 5]:
        return token_logprobs(X, t)

    @ml_function(target="b200")
    def twice(A: Tensor[f32, 64, 64], W: Tensor[f32, 64, 64]) -> Tensor[f32, 64, 64]:
        return (A @ W) @ W

    rng = np.random.default_rng(1)
    X, W = (rng.standard_normal((n, 64)).astype(np.float32) for n in (5, 64))
    x = torch.from_numpy(X).double()
    want = x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)
    assert (np.abs(norm(X) - want.numpy()) <= NORM_F32 * np.abs(want.numpy()) + 2.0 ** -149).all()
    got = score(X, np.array([3, 0, -1, 63, 64], np.int32))
    logs = torch.log_softmax(x, 1)
    assert np.abs(got[[0, 1, 3]] - [logs[0, 3], logs[1, 0], logs[3, 63]]).max() <= 2.0 ** -18
    assert got[2] == 0 and np.isnan(got[4])
    register_weights(W, bits=4, group=64)
    try:
        left = twice(W, W)
    finally:
        release_weights(W)
    D = serving.quantize_w4(torch.from_numpy(W).to(cuda), group=64).dequantize().cpu().double()
    w = torch.from_numpy(W).double()
    inner = w @ D
    # 2^-18 of the sum of absolute products in each layer, carried through the second
    room = 2.0 ** -18 * (w.abs() @ D.abs() @ D.abs() + inner.abs() @ D.abs())
    assert (np.abs(left - (inner @ D).numpy()) <= room.numpy()).all()


# ------------------------------------------------- offsets past 2^31 elements

@pytest.fixture
def room(cuda):
    """Fresh memory before and after a test of some GB."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M,N,quant", [(540000, 4096, True), (540000, 4091, True),
                                       (70000, 32768, False)])
def test_rms_norm_far_rows(cuda, room, M, N, quant):
    x = torch.zeros(M, N, dtype=BF16, device=cuda)
    last = [0, M // 2, M - 2, M - 1]
    x[last] = rand(cuda, 1, 4, N).bfloat16()
    w = (rand(cuda, 2, N) * 0.1 + 1).bfloat16()
    out = serving.rms_norm(x, w, quant="e4m3", group=128) if quant else serving.rms_norm(x, w)
    synced()
    want = norm_formula(x[last], 1e-6) * w.double()
    if not quant:
        room = half_step(want, BF16) + NORM_F32 * want.abs()
        assert ((out[last].double() - want).abs() <= room).all() and (out[M - 3] == 0).all()
        return
    codes, scales = out
    assert (scales[M - 3] == 1).all() and (scales[M // 2 + 1] == 1).all()
    assert (codes[M - 3].float() == 0).all()
    per = scales[last].double().repeat_interleave(128, 1)[:, :N]
    for i, g0 in enumerate(range(0, N, 128)):
        most = want[:, g0:g0 + 128].abs().amax(1) / 448
        assert ((scales[last, i].double() - most).abs() <= 2 * NORM_F32 * most).all()
    # half a step of e4m3 of the value, or near 0 of its smallest one
    step = torch.maximum(want.abs() * 2.0 ** -4, per * 2.0 ** -10)
    value = codes[last].double() * per
    assert ((value - want).abs() <= step * (1 + 2.0 ** -10) + 4 * NORM_F32 * want.abs()).all()


def test_token_logprobs_far_rows(cuda, room):
    T, V = 20000, 131072
    logits = torch.zeros(T, V, dtype=F16, device=cuda)
    last = [0, T // 2, T - 1]
    logits[last] = (rand(cuda, 1, 3, V) * 3).half()
    tokens = torch.arange(T, dtype=torch.int32, device=cuda)
    out = serving.token_logprobs(logits, tokens, top=5)
    synced()
    for i, row in enumerate(last):
        x = logits[row].double()
        order = torch.sort(x, descending=True, stable=True)
        lse = torch.logsumexp(x, 0)
        assert torch.equal(out.top_tokens[row].long(), order.indices[:5])
        # as for rows of one thread's tokens, with 512 logits a thread
        assert ((out.top_logprobs[row].double() - (order.values[:5] - lse)).abs() <= 2.0 ** -13).all()
        assert abs(out.logprobs[row].double() - (x[row] - lse)) <= 2.0 ** -13
    assert (out.top_tokens[T - 2] == torch.arange(5, device=cuda)).all()


@pytest.mark.parametrize("M", [5, 17])
def test_dense_w4_far_rows(cuda, room, M):
    """Rows of X and of Y that lie 2^32 bytes apart and more."""
    K, N, far = 256, 130, (1 << 32) // (M - 1) + 64
    w = serving.quantize_w4(rand(cuda, 1, K, N), group=64)
    x = torch.empty((M - 1) * far + K, dtype=BF16, device=cuda).as_strided((M, K), (far, 1))
    y = torch.empty((M - 1) * far + N, dtype=BF16, device=cuda).as_strided((M, N), (far, 1))
    x.copy_(rand(cuda, 2, M, K))
    want = serving.dense_w4(x.contiguous(), w)
    serving.dense_w4(x, w, out=y)
    synced()
    assert torch.equal(y, want)
