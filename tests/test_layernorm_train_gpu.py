"""LayerNorm for training: the forward with statistics and the backward against 64 bits.

Tolerances count roundings of u = 2^-24 (f32) on the terms they are made on.  A row sum is made of 8 sequential
additions a thread and 10 levels (one more addition for each 1024 elements of a long row), so a sum over N terms is within
(20 + N / 1024) u of the sum of their sizes, and every result has fewer than 12 further roundings: k = 32 + N / 1024 of
the sizes of its terms.  bf16 results have half a step, 2^-8 of the value, more."""
import numpy as np
import pytest

import oracle
from gpu_util import bf16_round, dev, rng, to_gpu, torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def ops():
    dev()
    from teenygrad_b200 import ops as o
    return o


def cast_of(dtype):
    return bf16_round if dtype == torch.bfloat16 else (lambda a: np.asarray(a, np.float32))


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, ref, bound, bf16=False, what=""):
    got = f64(got)
    bound = np.broadcast_to(np.asarray(bound) + (2.0 ** -8 * np.abs(ref) if bf16 else 0), ref.shape)
    bad = np.abs(got - ref) > bound
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}: " \
                          f"{got[bad][0]} against {ref[bad][0]}, bound {bound[bad][0]:.2e}"


def inputs(M, N, dtype, seed=0, offset=0.5):
    r = rng(seed * 1000 + M + N)
    c = cast_of(dtype)
    x = c(r.standard_normal((M, N)) * r.uniform(0.5, 2, (M, 1)) + offset * r.standard_normal((M, 1)))
    return x, c(r.uniform(0.5, 1.5, N)), c(r.standard_normal(N)), c(r.standard_normal((M, N)))


def check_fwd(x, w, b, y, mean, rstd, eps, bf16):
    N = x.shape[1]
    k = 32 + N / 1024
    x, w, b = (np.asarray(a, np.float64) for a in (x, w, b))
    mu = x.mean(1, keepdims=True)
    size = np.abs(x).mean(1, keepdims=True)
    var = ((x - mu) ** 2).mean(1, keepdims=True)
    rs = 1 / np.sqrt(var + eps)
    xh = (x - mu) * rs
    close(mean, mu[:, 0], k * U * size[:, 0], what="mean")
    # the mean's own error enters the variance squared
    close(rstd, rs[:, 0], (k * U * rs + rs ** 3 * (k * U * size) ** 2)[:, 0], what="rstd")
    close(y, xh * w + b, k * U * (np.abs(w) * (np.abs(xh) + rs * size) + np.abs(b)), bf16, "y")


def check_bwd(dy, x, w, mean, rstd, got, bf16, dw0=0.0, db0=0.0):
    M, N = x.shape
    k = 32 + N / 1024
    dy, x, w, mu, rs = (np.asarray(a, np.float64) for a in (dy, x, w, mean, rstd))
    mu, rs = mu[:, None], rs[:, None]
    xh, a = (x - mu) * rs, dy * w
    c1, c2 = a.mean(1, keepdims=True), (a * xh).mean(1, keepdims=True)
    dx, dw, db = got
    size = np.abs(a) + np.abs(a).mean(1, keepdims=True) + np.abs(xh) * np.abs(a * xh).mean(1, keepdims=True)
    close(dx, rs * (a - c1 - xh * c2), k * U * rs * size, bf16, "dx")
    # columns: M / 148 rows a thread at least, 8 warps, 16 lanes of the CTAs' sums (at most 592 of them)
    kc = 16 + M / 148 + 8 + 16 + 592 / 16
    close(dw, dw0 + (dy * xh).sum(0), kc * U * (np.abs(dw0) + np.abs(dy * xh).sum(0)), what="dw")
    close(db, db0 + dy.sum(0), kc * U * (np.abs(db0) + np.abs(dy).sum(0)), what="db")


SIZES = [(1, 1), (3, 1), (5, 2), (7, 8), (1, 256), (9, 255), (128, 256), (300, 264), (17, 1000), (33, 1024), (5, 1025),
         (40, 2048), (1300, 2048), (6, 2051), (19, 4096), (3, 5003), (11, 8192), (2, 8191), (4, 8193), (35, 8200),
         (3, 16384), (2, 40001), (70000, 8), (5000, 37)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N", SIZES)
def test_forward_and_backward(dtype, M, N):
    o, bf16 = ops(), dtype == torch.bfloat16
    x, w, b, dy = inputs(M, N, dtype)
    gx, gw, gb, gdy = (to_gpu(a, dtype) for a in (x, w, b, dy))
    y, mean, rstd = o.layer_norm(gx, gw, gb, 1e-5, return_stats=True)
    assert y.dtype == dtype and mean.shape == rstd.shape == (M,)
    check_fwd(x, w, b, y, mean, rstd, 1e-5, bf16)
    got = o.layer_norm_backward(gdy, gx, gw, mean, rstd)
    assert got[0].dtype == dtype and got[1].dtype == got[2].dtype == torch.float32
    check_bwd(dy, x, w, f64(mean), f64(rstd), got, bf16)
    for a, c in zip(got, o.layer_norm_backward(gdy, gx, gw, mean, rstd)):   # the same bits again
        assert torch.equal(a, c)


@pytest.mark.parametrize("N", [264, 9001])
def test_inputs_at_odd_addresses(N):
    o, M = ops(), 13
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, dy = inputs(M, N, dtype, seed=1)

        def odd(a):
            t = torch.empty(a.size + 1, device="cuda", dtype=dtype)[1:].view(a.shape)
            return t.copy_(torch.from_numpy(np.ascontiguousarray(a)))

        gx, gw, gb, gdy = odd(x), odd(w), odd(b), odd(dy)
        y, mean, rstd = o.layer_norm(gx, gw, gb, return_stats=True)
        check_fwd(x, w, b, y, mean, rstd, 1e-5, dtype == torch.bfloat16)
        check_bwd(dy, x, w, f64(mean), f64(rstd), o.layer_norm_backward(gdy, gx, gw, mean, rstd), dtype == torch.bfloat16)


def test_forward_matches_the_inference_forward_and_the_oracle():
    o = ops()
    x, w, b, _ = inputs(48, 768, torch.float32, seed=2)
    y, _, _ = o.layer_norm(to_gpu(x), to_gpu(w), to_gpu(b), 1e-5, return_stats=True)
    ref = oracle.layernorm(x, w, b, 1e-5)
    ref = np.asarray(ref[0] if isinstance(ref, tuple) else ref, np.float64)
    np.testing.assert_allclose(f64(y), ref, rtol=0, atol=32 * U * 20)
    np.testing.assert_allclose(f64(o.layer_norm(to_gpu(x), to_gpu(w), to_gpu(b), 1e-5)), f64(y), rtol=0, atol=64 * U * 20)


def test_mean_far_from_zero_and_constant_rows():
    o = ops()
    r = rng(5)
    x = (r.standard_normal((6, 512)) * 1e-2 + 1000).astype(np.float32)
    x[1], x[2] = 7.0, 0.0
    w, b = np.ones(512, np.float32), np.zeros(512, np.float32)
    y, mean, rstd = o.layer_norm(to_gpu(x), to_gpu(w), to_gpu(b), 1e-5, return_stats=True)
    check_fwd(x, w, b, y, mean, rstd, 1e-5, False)


def test_gradient_sums_accumulate():
    o = ops()
    for M in (3, 100, 2000):   # one CTA, and more
        sums_accumulate(o, M)


def sums_accumulate(o, M):
    x, w, _, dy = inputs(M, 520, torch.bfloat16, seed=3)
    r = rng(1)
    dw0, db0 = r.standard_normal(520).astype(np.float32), r.standard_normal(520).astype(np.float32)
    g = [to_gpu(a, torch.bfloat16) for a in (dy, x, w)]
    mean, rstd = to_gpu(x.mean(1)), to_gpu(1 / x.std(1))
    dw, db = to_gpu(dw0), to_gpu(db0)
    got = o.layer_norm_backward(*g, mean, rstd, dw, db)
    assert got[1] is dw and got[2] is db
    check_bwd(dy, x, w, f64(mean), f64(rstd), got, True, dw0.astype(np.float64), db0.astype(np.float64))


def test_no_rows():
    o = ops()
    x, w = torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda")
    y, mean, rstd = o.layer_norm(x, w, w, return_stats=True)
    assert y.shape == (0, 64) and mean.numel() == rstd.numel() == 0
    dx, dw, db = o.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    dw, db = torch.full_like(w, 3.0), torch.full_like(w, 4.0)
    o.layer_norm_backward(x, x, w, mean, rstd, dw, db)
    assert (dw == 3).all() and (db == 4).all()


def test_a_bad_row_stays_in_its_row():
    o = ops()
    x, w, b, dy = inputs(9, 300, torch.float32, seed=4)
    gx, gw, gb, gdy = (to_gpu(a) for a in (x, w, b, dy))
    y0, mean, rstd = o.layer_norm(gx, gw, gb, return_stats=True)
    dx0, _, db0 = o.layer_norm_backward(gdy, gx, gw, mean, rstd)
    gx[4, 7] = float("inf")
    gx[5, 299] = float("nan")
    y, mean, rstd = o.layer_norm(gx, gw, gb, return_stats=True)
    dx, dw, db = o.layer_norm_backward(gdy, gx, gw, mean, rstd)
    good = [0, 1, 2, 3, 6, 7, 8]
    assert torch.equal(y[good], y0[good]) and torch.equal(dx[good], dx0[good]) and torch.equal(db, db0)
    assert y[4:6].isnan().all() and dx[4:6].isnan().all() and dw.isnan().all()


def test_leading_dimensions():
    o = ops()
    x, w, b, dy = inputs(24, 96, torch.float32, seed=6)
    gx, gw, gb, gdy = (to_gpu(a) for a in (x, w, b, dy))
    y, mean, rstd = o.layer_norm(gx.view(2, 3, 4, 96), gw, gb, return_stats=True)
    y2, mean2, rstd2 = o.layer_norm(gx, gw, gb, return_stats=True)
    assert y.shape == (2, 3, 4, 96) and torch.equal(y.view(24, 96), y2) and torch.equal(mean, mean2)
    dx, dw, db = o.layer_norm_backward(gdy.view(2, 3, 4, 96), gx.view(2, 3, 4, 96), gw, mean, rstd)
    dx2, dw2, db2 = o.layer_norm_backward(gdy, gx, gw, mean2, rstd2)
    assert dx.shape == (2, 3, 4, 96) and torch.equal(dx.view(24, 96), dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("N", [40, 700])
def test_gradient_against_differences(N):
    """dx, dw and db against central differences of sum(dy * norm(x)), itself in 64 bits."""
    o = ops()
    x, w, b, dy = inputs(3, N, torch.float32, seed=7)
    gx, gw = to_gpu(x), to_gpu(w)
    _, mean, rstd = o.layer_norm(gx, gw, to_gpu(b), return_stats=True)
    dx, dw, db = (f64(t) for t in o.layer_norm_backward(to_gpu(dy), gx, gw, mean, rstd))

    def loss(x, w, b):
        d = x - x.mean(1, keepdims=True)
        return (dy * (d / np.sqrt((d * d).mean(1, keepdims=True) + 1e-5) * w + b)).sum()

    args = [np.asarray(a, np.float64) for a in (x, w, b)]
    r, h = rng(0), 1e-4
    for k, grad in enumerate((dx, dw, db)):
        for _ in range(8):
            at = tuple(r.integers(0, s) for s in args[k].shape)
            hi, lo = [a.copy() for a in args], [a.copy() for a in args]
            hi[k][at] += h
            lo[k][at] -= h
            # h^2 of a third derivative of some |dy| N^0, and 64 bits' own cancellation: 1e-6 of values of order 1
            assert abs((loss(*hi) - loss(*lo)) / (2 * h) - grad[at]) < 1e-5 * (1 + abs(grad[at]))


def test_offsets_past_32_bits():
    o = ops()
    # 2.15e9 elements, in the long rows' kernels and in the registers'; a column is summed in 60 parts at least
    for M, N in ((262152, 8200), (1050000, 2048)):
        x = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
        g = torch.Generator(device="cuda").manual_seed(0)
        for part in x.split(65536):
            part.copy_(torch.randn(part.shape, device="cuda", generator=g))
        w = torch.rand(N, device="cuda", generator=g).bfloat16()
        b = torch.zeros_like(w)
        y, mean, rstd = o.layer_norm(x, w, b, return_stats=True)
        few = x[-3:].clone()
        y2, mean2, rstd2 = o.layer_norm(few, w, b, return_stats=True)
        assert torch.equal(y[-3:], y2) and torch.equal(mean[-3:], mean2) and torch.equal(rstd[-3:], rstd2)
        del y
        dx, dw, db = o.layer_norm_backward(x, x, w, mean, rstd)
        dx2, _, _ = o.layer_norm_backward(few, few, w, mean2, rstd2)
        assert torch.equal(dx[-3:], dx2)
        want = torch.zeros(N, device="cuda", dtype=torch.float64)
        size = torch.zeros_like(want)
        for part in x.split(65536):
            want += part.double().sum(0)
            size += part.double().abs().sum(0)
        assert ((db.double() - want).abs() <= (100 + M / 60) * U * size).all()
        del x, dx


def test_on_another_stream_and_replayed():
    o = ops()
    x, w, b, dy = (to_gpu(a, torch.bfloat16) for a in inputs(200, 1024, torch.bfloat16, seed=8))
    want = o.layer_norm(x, w, b, return_stats=True)
    wantb = o.layer_norm_backward(dy, x, w, *want[1:])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = o.layer_norm(x, w, b, return_stats=True)
        gotb = o.layer_norm_backward(dy, x, w, *got[1:])
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want + wantb, got + gotb))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = o.layer_norm(x, w, b, return_stats=True)
        out = o.layer_norm_backward(dy, x, w, mean, rstd)
    x.copy_(x.flip(0))
    dy.copy_(dy.flip(0))
    want = o.layer_norm(x, w, b, return_stats=True)
    wantb = o.layer_norm_backward(dy, x, w, *want[1:])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[0]) and all(torch.equal(p, q) for p, q in zip(wantb, out))


def test_refusals():
    o = ops()
    from teenygrad_b200 import TeenyError
    M = 200
    x, w = torch.ones(M, 8, device="cuda"), torch.ones(8, device="cuda")
    mean, rstd = torch.ones(M, device="cuda"), torch.ones(M, device="cuda")
    bad = [
        lambda: o.layer_norm(x, w[:4], w, return_stats=True),
        lambda: o.layer_norm(x, w, w.bfloat16(), return_stats=True),
        lambda: o.layer_norm(x.half(), w.half(), w.half(), return_stats=True),
        lambda: o.layer_norm(x.t(), w, w, return_stats=True),
        lambda: o.layer_norm(x[:, :0].contiguous(), w[:0], w[:0], return_stats=True),
        lambda: o.layer_norm(x[0, 0], w[:1], w[:1], return_stats=True),
        lambda: o.layer_norm_backward(x[:, :0].contiguous(), x[:, :0].contiguous(), w[:0], mean, rstd),
        lambda: o.layer_norm_backward(x[:2], x, w, mean, rstd),
        lambda: o.layer_norm_backward(x.bfloat16(), x, w, mean, rstd),
        lambda: o.layer_norm_backward(x, x, w, mean[:3], rstd),
        lambda: o.layer_norm_backward(x, x, w, mean.double(), rstd),
        lambda: o.layer_norm_backward(x, x, w, mean, rstd, dw=torch.zeros(8, device="cuda")),
        lambda: o.layer_norm_backward(x, x, w, mean, rstd, torch.zeros(7, device="cuda"), torch.zeros(7, device="cuda")),
    ]
    for call in bad:
        with pytest.raises(TeenyError):
            call()
    buf = torch.zeros(8, device="cuda")
    with pytest.raises(TeenyError):   # the two sums in one place
        o.layer_norm_backward(x, x, w, mean, rstd, buf, buf)
    from teenygrad_b200 import lib
    ctx = o.context()
    args = (ctx, 0, x.data_ptr(), x.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr())
    ws = torch.empty(1 << 20, device="cuda", dtype=torch.uint8)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    tail = (dw.data_ptr(), db.data_ptr(), 0, M, 8)
    l = lib()
    assert l.tb_layernorm_bwd(*args, dx.data_ptr(), *tail, ws.data_ptr(), 16) == 1          # too small a workspace
    assert l.tb_layernorm_bwd(*args, dx.data_ptr(), *tail, ws.data_ptr() + 4, 1 << 19) == 3  # at an odd address
    assert l.tb_layernorm_bwd(*args, x.data_ptr(), *tail, ws.data_ptr(), 1 << 20) == 1       # in place
    assert l.tb_layernorm_fwd_train(ctx, 0, x.data_ptr(), w.data_ptr(), w.data_ptr(), x.data_ptr(), mean.data_ptr(),
                                    rstd.data_ptr(), M, 8, 1e-5) == 1
    assert l.tb_layernorm_fwd_train(ctx, 0, x.data_ptr(), w.data_ptr(), w.data_ptr(), dx.data_ptr(), mean.data_ptr(),
                                    rstd.data_ptr(), M, 0, 1e-5) == 2
    assert b"overlap" not in l.tb_last_error(ctx)
    # between two floats; statistics in y; sums in the workspace
    assert l.tb_layernorm_fwd_train(ctx, 0, x.data_ptr(), w.data_ptr() + 2, w.data_ptr(), dx.data_ptr(), mean.data_ptr(),
                                    rstd.data_ptr(), M, 8, 1e-5) == 3
    assert l.tb_layernorm_fwd_train(ctx, 0, x.data_ptr(), w.data_ptr(), w.data_ptr(), dx.data_ptr(), dx.data_ptr(),
                                    rstd.data_ptr(), M, 8, 1e-5) == 1
    assert l.tb_layernorm_bwd(*args, dx.data_ptr(), ws.data_ptr(), db.data_ptr(), 0, M, 8, ws.data_ptr(), 1 << 20) == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("M,N,odd", [(33, 264, True), (1000, 264, True), (1000, 2048, True), (47, 9001, True), (100, 8193, False),
                                     (50, 12001, False), (40, 16384, True), (40, 16384, False)])
def test_element_by_element_backward_in_several_splits(M, N, odd, accumulate, dtype):
    """Tensors at odd addresses and long odd rows with more rows than one split takes: the partial sums stay in a
    workspace of the size that is asked for, which is full of what another kernel left."""
    import ctypes
    o = ops()
    from teenygrad_b200._lib import check, lib
    bf16 = dtype == torch.bfloat16
    x, w, _, dy = inputs(M, N, dtype, seed=9)
    r = rng(2)

    def at(a):
        lead = 1 if odd else 0
        t = torch.empty(a.size + lead, device="cuda", dtype=dtype)[lead:].view(a.shape)
        return t.copy_(torch.from_numpy(np.ascontiguousarray(a)))

    gx, gw, gdy = at(x), at(w), at(dy)
    mean, rstd = to_gpu(x.mean(1)), to_gpu(1 / np.sqrt(x.astype(np.float64).var(1) + 1e-5))
    dw0, db0 = (r.standard_normal(N).astype(np.float32) for _ in range(2))
    dw, db, dx = to_gpu(dw0), to_gpu(db0), torch.empty_like(gx)
    code, need = 1 if bf16 else 0, ctypes.c_size_t(0)
    assert lib().tb_workspace_bytes(13, code, (ctypes.c_int64 * 2)(M, N), 2, ctypes.byref(need)) == 0
    assert need.value >= 2 * 2 * N * 4
    buf = torch.full((need.value + 512,), 0xFF, device="cuda", dtype=torch.uint8)   # NaN, as f32
    ctx = o.context()
    check(ctx, lib().tb_layernorm_bwd(ctx, code, gdy.data_ptr(), gx.data_ptr(), gw.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                      dx.data_ptr(), dw.data_ptr(), db.data_ptr(), accumulate, M, N, buf.data_ptr() + 256,
                                      need.value))
    zero = np.zeros(N)
    check_bwd(dy, x, w, f64(mean), f64(rstd), (dx, dw, db), bf16, *((dw0.astype(np.float64), db0.astype(np.float64)) if accumulate
                                                                     else (zero, zero)))
    assert bool((buf[:256] == 0xFF).all() and (buf[-256:] == 0xFF).all())
