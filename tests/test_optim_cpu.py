"""The 8-bit moments' definition (in the restatement that the GPU tests hold the kernel to), and refusals that need no GPU."""
import ctypes

import numpy as np
import pytest

import optim_util as u

torch = pytest.importorskip("torch")

import teenygrad_b200 as tg  # noqa: E402
from teenygrad_b200 import ops  # noqa: E402


def test_e4m3_values_are_torchs():
    code = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(code).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(u.e4m3(code), want)


def test_random_bits_are_uniform_and_independent():
    n = 1 << 18
    a, b, c = u.random_bits(1, 1, 0, n), u.random_bits(1, 2, 0, n), u.random_bits(1, 1, 1, n)
    # the mean of a fair bit over 2^18 has a deviation of sqrt(1/4 / 2^18) = 2^-10; 6 of them
    for x in (a, b, c, a ^ b, a ^ c, a ^ np.roll(a, 1), a ^ np.roll(a, 256), (a ^ (a >> np.uint32(16))) << np.uint32(16)):
        bits = [((x >> np.uint32(k)) & np.uint32(1)).mean() for k in range(32)]
        assert all(abs(m - 0.5) < 6 * 2.0 ** -10 for m in bits if m)
        assert sum(not m for m in bits) in (0, 16)
    h = np.bincount(a >> np.uint32(24), minlength=256)
    assert ((h - n / 256) ** 2 / (n / 256)).sum() < 255 + 6 * np.sqrt(2 * 255)
    assert len(np.unique(u.random_bits(7, 3, 2, n))) == n   # one tensor's words are all different
    # past 2^32 elements the high word counts
    far = u.random_bits(1, 1, 0, 16, first=1 << 32)
    assert not np.array_equal(far, a[:16])


@pytest.mark.parametrize("size", [1.0, 1e-30, 3e20])
def test_rounding_has_the_values_mean(size):
    r = np.random.default_rng(5)
    x = (r.standard_normal(256) * 10.0 ** r.uniform(-7, 0, 256) * size).astype(np.float32)
    total, square, T = np.zeros(256), np.zeros(256), 4000
    for t in range(T):
        code, e = u.encode(x, u.random_bits(3, t + 1, 0, 256) & np.uint32(0xFFFF), False)
        v = u.held(code, e).astype(np.float64)
        total += v
        square += v * v
    mean = total / T
    # the step of the grid at x bounds a draw's deviation by half of it; 6 deviations of the mean, and the 2^-17
    # that 16 bits leave
    scale = 2.0 ** (int(e[0]) - 127)
    y = np.maximum(np.abs(x).astype(np.float64) / scale, 2.0 ** -6)
    step = np.exp2(np.floor(np.log2(y)) - 3) * scale
    assert np.all(np.abs(mean - x) <= step * (0.5 * 6 / np.sqrt(T) + 2.0 ** -16))
    # a value never leaves the two codes around it
    assert np.all(np.sqrt(np.maximum(square / T - mean * mean, 0)) <= step)


def test_codes_of_the_edges():
    def one(x, bits, root=False):
        a = np.zeros(256, np.float32)
        a[0], a[1] = 255.0, x      # the exponent puts 255 at 255
        code, e = u.encode(a, np.full(256, bits, np.uint32), root)
        assert e[0] == 127
        return float(u.e4m3(code)[1])

    assert one(240.0, 0xFFFF) == 240.0 and one(-240.0, 0) == -240.0   # what the grid holds stays
    assert one(241.0, 0xFFFF) == 256.0 and one(241.0, 0) == 240.0
    assert one(2.0 ** -10, 0) == 0.0 and one(2.0 ** -10, 0xFFFF) == 2.0 ** -9
    assert one(2.0 ** -30, 0, root=True) == 2.0 ** -9                 # a root above zero stays above it
    assert one(0.0, 0xFFFF, root=True) == 0.0
    zero, e = u.encode(np.zeros(300, np.float32), np.full(300, 0xFFFF, np.uint32), True)
    assert not zero.any() and not e.any() and len(e) == 2
    bad = np.zeros(256, np.float32)
    bad[:4] = np.inf, -np.inf, np.nan, 1.0
    code, e = u.encode(bad, np.zeros(256, np.uint32), False)
    assert np.isnan(u.e4m3(code[:3])).all() and u.held(code, e)[3] == 1.0


def test_root_follows_a_falling_gradient():
    """What rounding to nearest would not do: with beta2 = 0.999 the held root decays with the gradient."""
    n, T = 512, 2000
    r = np.random.default_rng(0)
    cm = cs = np.zeros(n, np.uint8)
    em = es = np.zeros(2, np.uint8)
    v = np.zeros(n)
    for t in range(1, 2 * T + 1):
        g = r.standard_normal(n) * (1.0 if t <= T else 0.01)
        cm, em, cs, es = u.adamw8_moments(g, cm, em, cs, es, 1, t, 0, 0.9, 0.999, 1.0)
        v = 0.999 * v + 0.001 * g * g
    s = u.held(cs, es).astype(np.float64)
    # a root's own deviation around the 32-bit one is some twenty percent; the mean over 512 has 1 %
    assert abs(np.mean(s / np.sqrt(v)) - 1) < 0.1


@pytest.mark.parametrize("low,high,tol", [(1.0, 8.0, 0.012), (4 * 2.0 ** -9, 8 * 2.0 ** -9, 0.03)])
def test_second_moment_is_high_by_the_roundings_variance(low, high, tol):
    """The root is rounded without bias, so its square is high by the rounding's variance.

    A step moves the root r by d = r (1 - b2) / 2 |g^2 / v - 1| from a code, and rounding back to that code or the next,
    a step of the grid away, has the variance d step.  Where b2 v + (1 - b2) g^2 + d step stays v on the average, v is
    1 / (1 - E|g^2 / v - 1| E[step / r] / 2) of the 32-bit one: for normal gradients E|g^2 / v - 1| = 4 phi(1) = 0.968, and
    for sizes spread evenly over a binade of normal codes E[step / r] = 1 / (16 ln 2) = 0.0902: 4.6 % high.  Where codes are
    k steps for k from 4 to 8 (the bottom of the range), E[step / r] = 1 / (8 ln 2): 9.6 %.  What is left out, the spread of
    v itself (0.09 and 0.17 of it, squared deviations) and d against a step, is under a third of these."""
    blocks, warm, T, b2 = 32, 400, 1000, 0.99
    n = blocks * 256
    r = np.random.default_rng(3)
    size = np.exp(r.uniform(np.log(low), np.log(high), n)) / 8   # the exponent puts 16 at 128
    first = np.arange(n) % 256 == 0
    cm = cs = np.zeros(n, np.uint8)
    em = es = np.zeros(blocks, np.uint8)
    v, held, true = np.zeros(n), 0.0, 0.0
    for t in range(1, warm + T + 1):
        g = np.where(first, 16.0, r.standard_normal(n) * size).astype(np.float32)
        cm, em, cs, es = u.adamw8_moments(g, cm, em, cs, es, 1, t, 0, 0.9, b2, 1.0)
        v = b2 * v + (1 - b2) * g.astype(np.float64) ** 2
        if t > warm:
            held += np.mean((u.held(cs, es).astype(np.float64) ** 2 / size ** 2)[~first])
            true += np.mean((v / size ** 2)[~first])
    inverse = 1 / (np.log(2) * 16) if low == 1.0 else 1 / (np.log(2) * 8)
    want = 1 / (1 - 4 * np.exp(-0.5) / np.sqrt(2 * np.pi) * inverse / 2)
    # 8160 elements with 10 independent spells each: 0.42 / sqrt(81600) is 0.15 % of chance
    assert abs(held / true - want) < tol, (held / true, want)


def test_refuses_cpu_tensors():
    x, w = torch.ones(4, 8), torch.ones(8)
    one = torch.ones(4)
    for call in (lambda: ops.layer_norm(x, w, w, return_stats=True),
                 lambda: ops.layer_norm_backward(x, x, w, one, one),
                 lambda: ops.grad_norm([x]),
                 lambda: ops.AdamW([x], [x])):
        with pytest.raises(tg.TeenyError):
            call()


def test_entry_points_refuse_without_a_context():
    l = tg.lib()
    assert l.tb_layernorm_fwd_train(None, 0, None, None, None, None, None, None, 1, 1, 1e-5) == 1
    assert l.tb_layernorm_bwd(None, 0, *[None] * 8, 0, 1, 1, None, 0) == 1
    assert l.tb_grad_norm(None, 0, None, None, 0, None, None, 1.0, None, 0) == 1
    h = ctypes.c_void_p(5)
    assert l.tb_adamw_create(None, 0, 0, 32, None, 0, ctypes.byref(h)) == 1 and not h.value
    assert l.tb_adamw_create(None, 0, 0, 32, None, 0, None) == 1
    assert l.tb_adamw_step(None, None) == 1
    assert l.tb_adamw_destroy(None) == 0


def test_workspaces_need_no_gpu():
    l = tg.lib()
    b = ctypes.c_size_t(0)

    def ask(op, *shape):
        return l.tb_workspace_bytes(op, 0, (ctypes.c_int64 * len(shape))(*shape), len(shape), ctypes.byref(b))

    assert ask(13, 1000, 64) == 0 and b.value >= 2 * 64 * 4 and b.value % (2 * 64 * 4) == 0
    assert ask(13, 0, 64) == 0 and b.value == 0
    assert ask(13, 1, 100000) == 0 and b.value == 0      # the sums of one CTA's rows are the results
    assert ask(13, 17, 100000) == 0 and b.value == 2 * 2 * 100000 * 4
    assert ask(13, 16) == 1 and ask(13, -1, 8) == 2 and ask(13, 8, 0) == 2 and ask(13, 1 << 31, 8) == 2
    assert ask(14, 3) == 0 and b.value > 0
    one = b.value
    assert ask(14, 1000) == 0 and b.value == 3 * one
    assert ask(14, -1) == 2 and ask(14) == 1
    out = ctypes.c_int64(0)
    assert l.tb_output_row_stride(13, 1, ctypes.c_int64(7), ctypes.byref(out)) == 0 and out.value == 7
