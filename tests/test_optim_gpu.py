"""The gradient norm and AdamW against 64 bits; the 8-bit moments bit for bit against their definition.  Tolerances: optim_util.bounds."""
import copy
import threading

import numpy as np
import pytest

import optim_util as u
from gpu_util import bf16_round, dev, rng, torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32, False), (F32, BF16, True), (F32, BF16, False), (BF16, BF16, False)]
SIZES = [1, 3, 255, 256, 257, 0, 2047, 2048, 2049, 5000, 70001]
B1, B2, EPS, WD, LR = 0.9, 0.999, 1e-8, 0.1, 3e-3


def ops():
    dev()
    from teenygrad_b200 import ops as o
    return o


def error():
    from teenygrad_b200 import TeenyError
    return TeenyError


def host(t):
    return t.detach().float().cpu().numpy()


def rounded(a, dtype):
    return bf16_round(a) if dtype == BF16 else np.asarray(a, np.float32)


def place(a, dtype, odd=False):
    """A tensor of a's values, at an address that no vector of four fits where `odd`, with guards on both sides."""
    n, lead = len(a), 33 if odd else 64
    buf = torch.full((n + lead + 64,), 77.0, device="cuda", dtype=F32).to(dtype)
    t = buf[lead:lead + n]
    t.copy_(torch.from_numpy(np.ascontiguousarray(a)).to(dtype) if n else t)
    return t, buf


def untouched(t, buf):
    lead = t.storage_offset()
    return bool((buf[:lead].float() == 77).all() and (buf[lead + t.numel():].float() == 77).all())


class Model:
    """Tensors of given sizes with their moments, on the device and on the host."""

    def __init__(self, sizes, pt, gt, copy, bits, seed=0, odd=False, spread=2.0):
        r = rng(seed)
        self.sizes, self.pt, self.gt, self.bits = sizes, pt, gt, bits
        wide = [10.0 ** r.uniform(-spread, 0) for _ in sizes]
        self.p = [rounded(r.standard_normal(n) * 0.1, pt) for n in sizes]
        self.g = [rounded(r.standard_normal(n) * w, gt) for n, w in zip(sizes, wide)]
        m = [(r.standard_normal(n) * 0.3 * w).astype(np.float32) for n, w in zip(sizes, wide)]
        v = [((r.standard_normal(n) ** 2 + 0.1) * w * w).astype(np.float32) for n, w in zip(sizes, wide)]
        self.made = [place(a, pt, odd) for a in self.p] + [place(a, gt, odd) for a in self.g]
        k = len(sizes)
        self.params, self.grads = [t for t, _ in self.made[:k]], [t for t, _ in self.made[k:]]
        self.copies = None
        if copy:
            c = [place(np.zeros(n), BF16, odd) for n in sizes]
            self.copies = [t for t, _ in c]
            self.made += c
        if bits == 32:
            self.m, self.v = m, v
            held = [place(a, F32, odd) for a in m + v]
            self.state = dict(m=[t for t, _ in held[:k]], v=[t for t, _ in held[k:]])
            self.made += held
        else:
            self.m = [u.encode(a, r.integers(0, 65536, len(a)), False) for a in m]
            self.s = [u.encode(np.sqrt(a), r.integers(0, 65536, len(a)), True) for a in v]

            def codes(a):
                buf = torch.full((len(a) + 64,), 77, device="cuda", dtype=torch.uint8)
                t = buf[(1 if odd else 32):][:len(a)]
                t.copy_(torch.from_numpy(a))
                self.made.append((t, buf))
                return t

            self.codes = dict(m=[codes(c) for c, _ in self.m], s=[codes(c) for c, _ in self.s],
                              m_exp=[codes(e) for _, e in self.m], s_exp=[codes(e) for _, e in self.s])
            self.state = {k: [t if k.endswith("exp") else t.view(torch.float8_e4m3fn) for t in ts]
                          for k, ts in self.codes.items()}

    def optimiser(self, step_count=0, **kw):
        args = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=self.bits, copies=self.copies,
                    state=self.state, step_count=step_count)
        return ops().AdamW(self.params, self.grads, **{**args, **kw})

    def check_codes(self, k, want):
        """Holds the codes of tensor k to adamw8_moments', bit for bit; the host takes them over."""
        cm, em, cs, es = want
        for name, code in (("m", cm), ("m_exp", em), ("s", cs), ("s_exp", es)):
            np.testing.assert_array_equal(self.codes[name][k].cpu().numpy(), code, err_msg=name)
        self.m[k], self.s[k] = (cm, em), (cs, es)

    def check(self, t, scale=1.0, seed=0, lr=LR, b1=B1, b2=B2, eps=EPS, wd=WD):
        """Holds the device's tensors after step t to the host's; the host takes them over."""
        scale = float(np.float32(scale))
        for k, n in enumerate(self.sizes):
            if self.bits == 32:
                m, v = self.m[k], self.v[k]
            else:
                m, v = u.held(*self.m[k]), u.held(*self.s[k]).astype(np.float64) ** 2
                self.check_codes(k, u.adamw8_moments(self.g[k], *self.m[k], *self.s[k], seed, t, k, b1, b2, scale))
            p, m1, v1, up, size, div = u.adamw64(self.p[k], self.g[k], m, v, t, lr, b1, b2, eps, wd, scale)
            bm, bp = u.bounds(self.p[k], up, size, div, p if self.pt == BF16 else None)
            got = host(self.params[k])
            if self.bits == 32:
                gm, gv = host(self.state["m"][k]), host(self.state["v"][k])
                assert np.all(np.abs(gm - m1) <= bm), n
                assert np.all(np.abs(gv - v1) <= 8 * u.U32 * v1), n
                self.m[k], self.v[k] = gm, gv
            assert np.all(np.abs(got - p) <= bp), (n, np.max(np.abs(got - p) / np.maximum(bp, 1e-300)))
            if self.copies is not None:
                np.testing.assert_array_equal(host(self.copies[k]), host(self.params[k].to(BF16)))
            self.p[k] = got
        assert all(untouched(t, buf) for t, buf in self.made)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("pt,gt,copy", TYPES)
def test_adamw_steps(pt, gt, copy, odd, bits):
    ops()
    m = Model(SIZES, pt, gt, copy, bits, odd=odd)
    o = m.optimiser(step_count=6, seed=9)
    scale = torch.tensor([0.37], device="cuda")
    o.step(grad_scale=scale)
    m.check(7, 0.37, seed=9)
    o.step(lr=1e-2)
    m.check(8, seed=9, lr=1e-2)
    assert o.step_count == 8


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_from_nothing(bits):
    """The first steps of a fresh optimiser, whose corrections divide by 1 - beta^t."""
    ops()
    m = Model([300, 1000], F32, F32, False, bits, seed=3)
    o = ops().AdamW(m.params, m.grads, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits, seed=5)
    if bits == 32:
        m.m, m.v = [np.zeros(n, np.float32) for n in m.sizes], [np.zeros(n, np.float32) for n in m.sizes]
        m.state = dict(m=o.m, v=o.v)
    else:
        zero = [(np.zeros(n, np.uint8), np.zeros(-(-n // 256), np.uint8)) for n in m.sizes]
        m.m, m.s = list(zero), list(zero)
        m.codes = dict(m=[t.view(torch.uint8) for t in o.m], s=[t.view(torch.uint8) for t in o.s], m_exp=o.m_exp,
                       s_exp=o.s_exp)
    for t in range(1, 6):
        o.step()
        m.check(t, seed=5)


@pytest.mark.parametrize("hyper", [dict(b1=0.0, b2=0.0), dict(b1=0.0, b2=0.99, eps=1e-3, wd=0.0),
                                   dict(b1=0.99, b2=0.95, lr=0.0, wd=0.5), dict(eps=0.0), dict(eps=1e-31, b2=0.5)])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_hyperparameters(bits, hyper):
    ops()
    h = dict(lr=LR, b1=B1, b2=B2, eps=EPS, wd=WD) | hyper
    m = Model([777], F32, F32, False, bits, seed=4)
    o = m.optimiser(lr=h["lr"], betas=(h["b1"], h["b2"]), eps=h["eps"], weight_decay=h["wd"], step_count=1000000)
    o.step()
    m.check(1000001, **h)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [48, 49, 440, 441, 1000])
def test_adamw_of_many_tensors(bits, n):
    ops()
    r = rng(n)
    m = Model([int(k) for k in r.integers(0, 600, n)], BF16, BF16, False, bits, seed=n)
    o = m.optimiser(step_count=2)
    o.step()
    m.check(3)


def test_adamw_8_bits_at_the_edges_of_the_range():
    """Gradients from the smallest numbers to the largest, zeros, and what is not finite, next to ordinary ones."""
    ops()
    m = Model([256 * 12], F32, F32, False, 8, seed=6)
    r = rng(1)
    g = r.standard_normal((12, 256)).astype(np.float32)
    scales = [1e-44, 1e-38, 1e-25, 1e-19, 1e-10, 1.0, 1e10, 1e17]
    with np.errstate(under="ignore"):
        for k, x in enumerate(scales):
            g[k] = g[k] * np.float32(x)
    g[8] = 0
    g[9] *= (np.float32(10.0) ** r.uniform(-12, 0, 256)).astype(np.float32)
    g[10, :5] = np.inf, -np.inf, np.nan, 3e38, -3e38
    m.g[0] = g.reshape(-1)
    m.grads[0].copy_(torch.from_numpy(m.g[0]))
    for name in ("m", "s", "m_exp", "s_exp"):   # the first eight blocks have seen nothing yet
        k = 8 * (1 if name.endswith("exp") else 256)
        m.codes[name][0][:k] = 0
    m.m[0][0][:8 * 256] = 0
    m.m[0][1][:8] = 0
    m.s[0][0][:8 * 256] = 0
    m.s[0][1][:8] = 0
    o = m.optimiser()
    for t in (1, 2, 3):
        o.step()
        m.check_codes(0, u.adamw8_moments(m.g[0], *m.m[0], *m.s[0], 0, t, 0, B1, B2, 1.0))
        p = host(m.params[0]).reshape(12, 256)
        bad = ~np.isfinite(p)
        assert bad[10, :3].all() and not np.delete(bad, 10, 0).any() and not bad[10, 5:].any()
    assert (host(m.state["s"][0]).reshape(12, 256)[10, 5:] < 256).all()


def test_adamw_8_bits_rounds_every_product():
    """Gradients of -9 times the held moment: the two products cancel to nothing only if each is rounded by itself."""
    ops()
    m = Model([256 * 64], F32, BF16, False, 8, seed=21)
    m.g[0] = bf16_round(-9 * u.held(*m.m[0]))
    m.grads[0].copy_(torch.from_numpy(m.g[0]))
    o = m.optimiser(step_count=10)
    o.step()
    m.check(11)
    assert (host(m.state["m"][0]) == 0).mean() > 0.2


def test_adamw_8_bits_where_the_root_is_at_a_border():
    """16 million roots, of which some hundred have their code decided by the last places of the square root."""
    ops()
    n = 1 << 24
    m = Model([n], F32, F32, False, 8, seed=31)
    o = m.optimiser(step_count=20)
    for t in (21, 22):
        o.step()
        m.check_codes(0, u.adamw8_moments(m.g[0], *m.m[0], *m.s[0], 0, t, 0, B1, B2, 1.0))


def test_adamw_8_bits_over_all_sizes():
    """A block for each power of two of the gradient, and the sizes within a block spread over forty more."""
    ops()
    k = 2 * 230
    m = Model([256 * k], F32, F32, False, 8, seed=16)
    r = rng(2)
    with np.errstate(under="ignore", over="ignore"):
        g = r.standard_normal((k, 256)) * 2.0 ** (np.arange(k)[:, None] // 2 - 150)
        g[1::2] *= 2.0 ** r.uniform(-40, 0, (k // 2, 256))
        m.g[0] = g.astype(np.float32).reshape(-1)
    m.grads[0].copy_(torch.from_numpy(m.g[0]))
    for name in m.codes:
        m.codes[name][0].zero_()
    m.m, m.s = [(np.zeros(256 * k, np.uint8), np.zeros(k, np.uint8))], [(np.zeros(256 * k, np.uint8), np.zeros(k, np.uint8))]
    o = m.optimiser(eps=1e-12)
    for t in (1, 2, 3, 4):
        o.step()
        m.check_codes(0, u.adamw8_moments(m.g[0], *m.m[0], *m.s[0], 0, t, 0, B1, B2, 1.0))
        if t == 2:   # a smaller gradient, so that the held moments count
            m.g[0] = (m.g[0] * np.float32(0.01)).astype(np.float32)
            m.grads[0].copy_(torch.from_numpy(m.g[0]))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_keeps_what_is_not_finite_to_itself(bits):
    ops()
    a, b = (Model([1000], F32, F32, False, bits, seed=8) for _ in range(2))
    b.grads[0][[3, 500]] = torch.tensor([float("inf"), float("nan")], device="cuda")
    for m in (a, b):
        m.optimiser(step_count=4).step()
    x, y = a.params[0].clone(), b.params[0].clone()
    assert not torch.isfinite(y[[3, 500]]).any()
    x[[3, 500]] = y[[3, 500]] = 0
    if bits == 8:   # such a block's operations are other ones: each of x and y is within some 32 half steps (u.bounds)
        assert torch.equal(x[512:], y[512:]) and ((x - y).abs() <= 64 * u.U32 * (x.abs() + 10 * LR)).all()
    else:
        assert torch.equal(x, y)


def test_adamw_of_nothing():
    o = ops()
    o.AdamW([], []).step()
    e = torch.empty(0, device="cuda")
    for bits in (32, 8):
        opt = o.AdamW([e], [e.clone()], state_bits=bits)
        opt.step()
        assert opt.step_count == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_captured_and_replayed(bits):
    ops()
    a, b = (Model([5000, 77], F32, BF16, True, bits, seed=2) for _ in range(2))
    lr, scale = torch.tensor([LR], device="cuda"), torch.ones(1, device="cuda")
    oa = a.optimiser(capturable=True, step_count=3)
    ob = b.optimiser(step_count=3)
    oa.step(lr=lr, grad_scale=scale)
    ob.step(grad_scale=scale)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step(lr=lr, grad_scale=scale)
    for k in range(3):
        lr.fill_(LR * (k + 1))
        scale.fill_(1.0 / (k + 1))
        for x, y in zip(a.grads, b.grads):
            x.mul_(0.5)
            y.mul_(0.5)
        graph.replay()
        ob.step(lr=lr, grad_scale=scale)
    torch.cuda.synchronize()
    assert oa.step_count == 7 == ob.step_count
    for x, y in zip(a.params + a.copies, b.params + b.copies):
        assert torch.equal(x, y)
    for name in a.state:
        for x, y in zip(a.state[name], b.state[name]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_adamw_on_another_stream():
    ops()
    a, b = (Model([100000], F32, F32, False, 32, seed=5) for _ in range(2))
    s = torch.cuda.Stream()
    oa, ob = a.optimiser(), b.optimiser()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            oa.step()
    for _ in range(3):
        ob.step()
    torch.cuda.synchronize()
    assert torch.equal(a.params[0], b.params[0])


def test_two_threads_on_streams_of_their_own():
    """Each thread's calls go to its own stream, whatever the other one does meanwhile."""
    o = ops()
    x = [torch.randn(300, 1000, device="cuda") for _ in range(2)]
    w = torch.rand(1000, device="cuda")
    models = [Model([30000, 77], F32, F32, False, bits, seed=7) for bits in (32, 8)]
    alone = [Model([30000, 77], F32, F32, False, bits, seed=7) for bits in (32, 8)]
    opts, refs = [m.optimiser() for m in models], [m.optimiser() for m in alone]
    want = [o.layer_norm(t, w, w, return_stats=True) for t in x]
    for r in refs:
        for _ in range(100):
            r.step()
    norms = [o.grad_norm([t]) for t in x]
    torch.cuda.synchronize()
    streams, bad = [torch.cuda.Stream() for _ in x], []

    def work(k):
        try:
            with torch.cuda.stream(streams[k]):
                for _ in range(100):
                    y = o.layer_norm(x[k], w, w, return_stats=True)
                    got = o.grad_norm([x[k]])
                    opts[k].step()
                    # read on this stream: what another stream wrote would be late
                    if not (all(torch.equal(a, b) for a, b in zip(y, want[k])) and torch.equal(got, norms[k])):
                        bad.append(k)
        except Exception as e:   # pragma: no cover - shown by the assertion
            bad.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad
    for m, a in zip(models, alone):
        assert all(torch.equal(p, q) for p, q in zip(m.params, a.params))


def test_adamw_refusals():
    o, E = ops(), error()

    def t(n=8, dtype=F32):
        return torch.zeros(n, device="cuda", dtype=dtype)

    p, g = t(), t()
    both = t(16)
    bad = [
        lambda: o.AdamW([p, p], [g, t()]),                                   # one parameter twice
        lambda: o.AdamW([both[:9], both[8:]], [t(9), t()]),                  # memory shared
        lambda: o.AdamW([p], [p]),                                           # a gradient that is written
        lambda: o.AdamW([p], [t(7)]),
        lambda: o.AdamW([p], []),
        lambda: o.AdamW([p.half()], [g.half()]),
        lambda: o.AdamW([p.bfloat16()], [g]),
        lambda: o.AdamW([p, t(8, BF16)], [g, t(8, BF16)]),
        lambda: o.AdamW([t(16)[::2]], [g]),
        lambda: o.AdamW([p.cpu()], [g]),
        lambda: o.AdamW([p], [g], copies=[t(8)]),
        lambda: o.AdamW([t(8, BF16)], [t(8, BF16)], copies=[t(8, BF16)]),
        lambda: o.AdamW([p], [g], state_bits=16),
        lambda: o.AdamW([p], [g], betas=(1.0, 0.9)),
        lambda: o.AdamW([p], [g], betas=(0.9, -0.1)),
        lambda: o.AdamW([p], [g], eps=float("nan")),
        lambda: o.AdamW([p], [g], step_count=-1),
        lambda: o.AdamW([p], [g], state=dict(m=[t(7)], v=[t()])),
        lambda: o.AdamW([p], [g], state=dict(m=[t(8, BF16)], v=[t(8, BF16)])),
        lambda: o.AdamW([p], [g], state_bits=8, state=dict(m=[t().to(torch.float8_e4m3fn)], s=[t().to(torch.float8_e4m3fn)],
                                                           m_exp=[t(2, torch.uint8)], s_exp=[t(1, torch.uint8)])),
        lambda: o.AdamW([p], [g]).step(lr=-1.0),
        lambda: o.AdamW([p], [g]).step(lr=float("nan")),
        lambda: o.AdamW([p], [g]).step(lr=torch.tensor([1.0])),
        lambda: o.AdamW([p], [g]).step(grad_scale=torch.ones(2, device="cuda")),
        lambda: o.AdamW([p], [g]).step(grad_scale=torch.ones(1, device="cuda", dtype=torch.float64)),
        lambda: o.grad_norm([p, g.bfloat16()]),
        lambda: o.grad_norm([p.half()]),
        lambda: o.grad_norm([t(16)[::2]]),
        lambda: o.grad_norm([p], max_norm=-1.0),
        lambda: o.grad_norm([p], max_norm=float("nan")),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(E):
            call()
            pytest.fail(f"call {k} was not refused")
    # a gradient may serve two parameters
    o.AdamW([t(), t()], [g, g]).step()
    # memory that moved
    q = t()
    opt = o.AdamW([q], [g])
    q.data = t()
    with pytest.raises(E, match="other memory"):
        opt.step()
    assert opt.step_count == 0
    with pytest.raises(E, match="has no v"):
        o.AdamW([p], [g], state=dict(m=[t()]))
    with pytest.raises(TypeError):
        copy.copy(opt)


def test_entry_points_refuse_bad_tables():
    import ctypes

    from teenygrad_b200 import lib
    ctx = ops().context()
    l, h = lib(), ctypes.c_void_p()
    t = [torch.zeros(64, device="cuda") for _ in range(4)]
    at = [x.data_ptr() for x in t]

    def create(row, n=1, p=0, g=0, bits=32):
        r = l.tb_adamw_create(ctx, p, g, bits, (ctypes.c_uint64 * len(row))(*row) if row else None, n, ctypes.byref(h))
        if not r:
            l.tb_adamw_destroy(h)
        return r

    good = at + [0, 0, 0, 64]
    assert create(good) == 0
    assert create(at[:3] + [0, 0, 0, 0, 64]) == 1            # no v
    assert create([at[0] + 2] + good[1:]) == 3               # between floats
    assert create(at + [0, 0, 0, (1 << 64) - 1]) == 2        # -1 elements
    assert create(at + [0, 0, 0, 1 << 40]) == 2              # more than are counted
    assert create(good, p=2) == 5 and create(good, p=1, g=0) == 5 and create(good, bits=16) == 5
    assert create(good, bits=8) == 1                         # no exponents
    assert create([], n=1) == 1 and create([], n=-1) == 1
    assert create([at[0], at[1], at[0], at[3], 0, 0, 0, 64]) == 1   # m where p is
    assert l.tb_grad_norm(ctx, 0, None, None, 1, at[0], None, 0.0, at[1], 256) == 1
    assert l.tb_grad_norm(ctx, 0, None, None, 0, at[0], None, 0.0, None, 0) == 1
    one, size = (ctypes.c_uint64 * 1)(at[0] + 1), (ctypes.c_int64 * 1)(8)
    ws = torch.empty(1 << 16, device="cuda", dtype=torch.uint8)
    assert l.tb_grad_norm(ctx, 0, one, size, 1, at[1], None, 0.0, ws.data_ptr(), 1 << 16) == 3
    size[0] = -1
    assert l.tb_grad_norm(ctx, 0, one, size, 1, at[1], None, 0.0, ws.data_ptr(), 1 << 16) == 2


def test_a_step_counted_on_the_host_is_not_captured():
    o, E = ops(), error()
    p, g = torch.zeros(8, device="cuda"), torch.ones(8, device="cuda")
    opt = o.AdamW([p], [g])
    opt.step()
    before = p.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(E, match="captured"):
            opt.step()
        p.add_(0)
    torch.cuda.synchronize()
    assert torch.equal(p, before) and opt.step_count == 1


# -------------------------------------------------------------- grad norm --
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sizes", [[1], [7], SIZES, [300001, 5, 1000], [13] * 60, [100] * 500, [3000] * 900])
def test_grad_norm(dtype, sizes):
    o, r = ops(), rng(len(sizes))
    g = [rounded(r.standard_normal(n) * 10.0 ** r.uniform(-3, 1), dtype) for n in sizes]
    ts = [place(a, dtype, odd=k % 2 == 1)[0] for k, a in enumerate(g)]
    want = np.sqrt(sum(float((a.astype(np.float64) ** 2).sum()) for a in g))
    # squares and 32 additions in f32: 33 half steps of the sum, half of that of the root, and its own rounding
    norm = o.grad_norm(ts)
    assert abs(float(norm) - want) <= 18 * u.U32 * want
    for top in (want / 3, want * 3, 0.0):
        norm2, scale = o.grad_norm(ts, max_norm=top)
        assert torch.equal(norm, norm2)
        assert abs(float(scale) - min(1.0, top / (want + 1e-6))) <= 20 * u.U32


def test_grad_norm_of_nothing_and_of_what_is_not_finite():
    o = ops()
    for ts in ([], [torch.empty(0, device="cuda")], [torch.zeros(100, device="cuda")]):
        norm, scale = o.grad_norm(ts, max_norm=1.0)
        assert float(norm) == 0 and float(scale) == 1
    g = torch.ones(5000, device="cuda")
    g[4999] = float("inf")
    norm, scale = o.grad_norm([g], max_norm=1.0)
    assert float(norm) == float("inf") and float(scale) == 0
    g[0] = float("nan")
    norm, scale = o.grad_norm([g], max_norm=1.0)
    assert torch.isnan(norm).all() and torch.isnan(scale).all()


def test_grad_norm_replayed_and_on_two_streams_at_once():
    o = ops()
    g = [torch.randn(200001, device="cuda"), torch.randn(3000000, device="cuda")]
    want = [o.grad_norm([x]) for x in g]
    streams = [torch.cuda.Stream() for _ in g]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(o.grad_norm([g[k]]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[k]) for k in (0, 1) for x in got[k])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, scale = o.grad_norm(g, max_norm=2.0)
    g[0].mul_(2)
    w = o.grad_norm(g, max_norm=2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(norm, w[0]) and torch.equal(scale, w[1])


# ------------------------------------------------------------- large, whole --
def test_offsets_past_32_bits():
    """A tensor of 2^32 + 300 elements: its last blocks against the same elements as a tensor of their own would be, but
    for the random bits, whose index has a high word."""
    o = ops()
    n, k = (1 << 32) + 300, 812
    p = torch.zeros(n, device="cuda", dtype=BF16)
    g = torch.zeros(n, device="cuda", dtype=BF16)
    r = rng(0)
    hp, hg = bf16_round(r.standard_normal(k)), bf16_round(r.standard_normal(k))
    p[-k:], g[-k:] = torch.from_numpy(hp).cuda(), torch.from_numpy(hg).cuda()
    norm = o.grad_norm([g])
    want = np.sqrt((hg.astype(np.float64) ** 2).sum())
    assert abs(float(norm) - want) <= 18 * u.U32 * want
    opt = o.AdamW([p], [g], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8, seed=3)
    opt.step()
    ref = o.AdamW([torch.from_numpy(hp).cuda().bfloat16()], [g[-k:].clone()], lr=LR, betas=(B1, B2), eps=EPS,
                  weight_decay=WD, state_bits=32)
    ref.step()
    # the update of a first step does not depend on the codes; its root is f32's root of the same square
    assert (p[-k:].float() - ref.params[0].float()).abs().max() <= 2.0 ** -7 * np.abs(hp).max()
    assert not p[:1000].any() and not opt.m[0].view(torch.uint8)[:-k].any()
    # elements before 2^32, and the block that starts there
    first = n - k
    bits = u.random_bits(3, 1, 0, k, first=first)
    with np.errstate(all="ignore"):
        m1 = hg * np.float32(1 - B1)
    pad = first % 256
    x = np.concatenate([np.zeros(pad, np.float32), m1])
    code, e = u.encode(x, np.concatenate([np.zeros(pad, np.uint32), bits & np.uint32(0xFFFF)]), False)
    np.testing.assert_array_equal(opt.m[0].view(torch.uint8)[-k:].cpu().numpy(), code[pad:])
    np.testing.assert_array_equal(opt.m_exp[0][-len(e):].cpu().numpy(), e)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step(bits):
    """linear -> layer norm -> mean square: the gradients of the operators in a row against automatic differentiation in 64
    bits, clipped and stepped."""
    o = ops()
    M, K, N = 64, 48, 40
    r = rng(11)
    x, w = (torch.from_numpy(a.astype(np.float32)).cuda() for a in (r.standard_normal((M, K)), r.standard_normal((N, K)) * 0.2))
    b, gamma, beta = (torch.from_numpy(a.astype(np.float32)).cuda() for a in
                      (r.standard_normal(N) * 0.1, 1 + 0.1 * r.standard_normal(N), 0.1 * r.standard_normal(N)))
    target = torch.from_numpy(r.standard_normal((M, N)).astype(np.float32)).cuda()
    params = [w, b, gamma, beta]
    grads = [torch.zeros_like(p) for p in params]
    opt = o.AdamW(params, grads, lr=1e-2, weight_decay=0.01, state_bits=bits)
    for t in range(1, 4):
        leaves = [p.double().requires_grad_() for p in params]
        h = x.double() @ leaves[0].t() + leaves[1]
        y = torch.nn.functional.layer_norm(h, (N,), leaves[2], leaves[3], 1e-5)
        want = torch.autograd.grad(((y - target.double()) ** 2).sum() / M, leaves)
        before = [host(p) for p in params]
        moments = [(host(opt.m[k]), host(opt.v[k])) if bits == 32 else
                   (u.held(opt.m[k].view(torch.uint8).cpu().numpy(), opt.m_exp[k].cpu().numpy()),
                    u.held(opt.s[k].view(torch.uint8).cpu().numpy(), opt.s_exp[k].cpu().numpy()).astype(np.float64) ** 2)
                   for k in range(4)]
        # the same with the operators
        h = o.linear(x, w, b)
        y, mean, rstd = o.layer_norm(h, gamma, beta, 1e-5, return_stats=True)
        dy = (y - target) * (2.0 / M)
        dh, dgamma, dbeta = o.layer_norm_backward(dy, h, gamma, mean, rstd)
        _, dw, db = o.linear_backward(x, w, dh)
        for dst, src, ref in zip(grads, (dw, db, dgamma, dbeta), want):
            dst.copy_(src.view(dst.shape))
            # sums of 64 terms of order |dy| |x| |rstd|, in f32: 1e-4 of the largest is 2^10 half steps
            assert (dst.double() - ref).abs().max() <= 1e-4 * ref.abs().max()
        norm, scale = o.grad_norm(grads, max_norm=0.5)
        opt.step(grad_scale=scale)
        c = float(scale)
        assert c < 1
        for k, p in enumerate(params):
            flat = lambda a: np.asarray(a).reshape(-1)  # noqa: E731
            ref, _, _, up, size, div = u.adamw64(flat(before[k]), flat(host(grads[k])), flat(moments[k][0]),
                                                 flat(moments[k][1]), t, 1e-2, 0.9, 0.999, 1e-8, 0.01, c)
            _, bp = u.bounds(flat(before[k]), up, size, div)
            assert np.all(np.abs(flat(host(p)) - ref) <= bp)


# ------------------------------------------------------- small numbers, eps --
def fresh(m):
    """Makes a Model's 8-bit moments those before the first step."""
    for name, held in (("m", m.m), ("s", m.s)):
        for k, n in enumerate(m.sizes):
            held[k] = (np.zeros(n, np.uint8), np.zeros(-(-n // 256), np.uint8))
            m.codes[name][k].zero_()
            m.codes[name + "_exp"][k].zero_()


@pytest.mark.parametrize("eps", [1e-10, 1e-12, 1e-15, 1e-20, 1e-25])
@pytest.mark.parametrize("pt,gt,copy", TYPES)
def test_adamw_8_bits_where_the_root_is_next_to_a_small_eps(pt, gt, copy, eps):
    """Second moments under 2^-126 in blocks of ordinary ones, whose roots are what an eps as small is added to."""
    ops()
    n = 512 * 5 + 100
    m = Model([n], pt, gt, copy, 8, seed=41)
    r = rng(3)
    g = r.standard_normal(n) * 1e-3
    tiny = r.random(n) < 0.3
    g[tiny] = (10.0 ** r.uniform(-19, np.log10(3e-18), n) * r.choice([-1, 1], n))[tiny]
    g[1024:1536] = 1e-3    # a unit of whole blocks that has none
    m.g[0] = rounded(g, gt)
    m.grads[0].copy_(torch.from_numpy(m.g[0]))
    for t in (1, 1000):
        fresh(m)
        m.optimiser(step_count=t - 1, eps=eps).step()
        zero = np.zeros(n)
        p, _, v, up, size, div = u.adamw64(m.p[0], m.g[0], zero, zero, t, LR, B1, B2, eps, WD, 1.0)
        _, bound = u.bounds(m.p[0], up, size, div, p if pt == BF16 else None)
        # under 2^-126 f32 has steps of 2^-149: half of one each for the square and its product, halved by the root
        bound = bound + np.abs(up) * 2.0 ** -149 / (2 * np.maximum(v, 2.0 ** -149))
        got = host(m.params[0])
        assert np.all(np.abs(got - p) <= bound), np.max(np.abs(got - p) / bound)
        m.check_codes(0, u.adamw8_moments(m.g[0], zero.astype(np.uint8), np.zeros(-(-n // 256), np.uint8), zero.astype(np.uint8),
                                          np.zeros(-(-n // 256), np.uint8), 0, t, 0, B1, B2, 1.0))
        m.p[0] = got


@pytest.mark.parametrize("eps", [1e-37, 1e-40, 1e-50])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_with_an_eps_under_f32s_normal_numbers(bits, eps):
    """What has no gradient and no moments is only decayed, for as long as eps is not 0."""
    ops()
    m = Model([1000], F32, F32, False, bits, seed=42)
    none = np.arange(1000) % 3 == 0
    m.g[0][none] = 0
    m.grads[0].copy_(torch.from_numpy(m.g[0]))
    if bits == 32:
        for held, name in ((m.m, "m"), (m.v, "v")):
            held[0][none] = 0
            m.state[name][0].copy_(torch.from_numpy(held[0]))
    else:
        for held, name in ((m.m, "m"), (m.s, "s")):
            held[0][0][none] = 0
            m.codes[name][0].copy_(torch.from_numpy(held[0][0]))
    o = m.optimiser(eps=eps, step_count=4)
    o.step()
    m.check(5, eps=eps)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1e-43, 1e-38, 1e-30, 1e-22, 1e-19, 1e-13, 1e12, 1e18, 1e25, 1e35])
def test_grad_norm_of_sizes_whose_squares_f32_does_not_hold(dtype, size):
    o, r = ops(), rng(7)
    small = size < 1
    # next to ordinary ones where those do not hide them: chunks of their own, and a few among zeros
    g = [r.standard_normal(20000) * size, np.where(r.random(9000) < 0.01, r.standard_normal(9000) * size, 0.0), np.zeros(8192)]
    if not small:
        g.append(r.standard_normal(5000))
    g = [rounded(a.astype(np.float32), dtype) for a in g]
    ts = [place(a, dtype, odd=k % 2 == 1)[0] for k, a in enumerate(g)]
    want = np.sqrt(sum(float((a.astype(np.float64) ** 2).sum()) for a in g))
    norm, scale = o.grad_norm(ts, max_norm=1.0)
    # as test_grad_norm has it; a result under 2^-126 has steps of 2^-149
    assert abs(float(norm) - want) <= 18 * u.U32 * want + 2.0 ** -150
    assert abs(float(scale) - min(1.0, 1 / (want + 1e-6))) <= 20 * u.U32 / max(want, 1.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_refuses_moments_that_were_given_other_memory(bits):
    ops(), error()
    m = Model([300, 77], F32, F32, False, bits, seed=43)
    for name in m.state:
        o = m.optimiser()
        o.step()
        before = host(m.params[1])
        kept = getattr(o, name)[1]
        old = kept.data
        kept.data = old.clone()            # as a restore may do
        with pytest.raises(error(), match="other memory"):
            o.step()
        kept.data = old
        o.step()                           # its own memory again
        getattr(o, name)[1] = old.clone()  # another tensor in its place
        with pytest.raises(error(), match="other memory"):
            o.step()
        assert o.step_count == 2
        assert not np.array_equal(host(m.params[1]), before)
    for name in ("params", "grads"):
        o = m.optimiser()
        getattr(o, name)[0] = getattr(o, name)[0].clone()
        with pytest.raises(error(), match="other memory"):
            o.step()


@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_is_not_counted(capturable):
    ops()
    a, b = (Model([300], F32, F32, False, 32, seed=44) for _ in range(2))
    o, ref = a.optimiser(capturable=capturable, step_count=5), b.optimiser(step_count=5)
    for x in (o, ref):
        x.step()
    o._hyper.eps = -1.0     # what the library refuses
    for _ in range(3):
        with pytest.raises(error()):
            o.step()
    assert o.step_count == 6
    o._hyper.eps = EPS
    for x in (o, ref):
        x.step()
    assert o.step_count == 7 and torch.equal(a.params[0], b.params[0])


def test_what_a_captured_step_reads_outlives_its_tensor():
    """A learning rate and a scale that are given other memory after the capture: the graph reads what it was made with."""
    ops()
    a, b = (Model([3000], F32, F32, False, 32, seed=45) for _ in range(2))
    lr, scale = torch.tensor([LR], device="cuda"), torch.tensor([0.25], device="cuda")
    oa, ob = a.optimiser(capturable=True), b.optimiser()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step(lr=lr, grad_scale=scale)
    lr.data, scale.data = torch.tensor([7.0], device="cuda"), torch.tensor([9.0], device="cuda")
    others = [torch.full((1,), 5.0, device="cuda") for _ in range(64)]   # would take freed memory
    for _ in range(2):
        graph.replay()
        ob.step(lr=LR, grad_scale=torch.tensor([0.25], device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(a.params[0], b.params[0]) and all(float(x) == 5 for x in others)
