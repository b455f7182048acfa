"""Cases of the training operators: LayerNorm with its gradient, the gradient norm of a whole model, and AdamW over
many tensors at once with moments in 32 bits or in 8.

`run` computes a case with elementary torch operations, or (where `own` is true) through teenygrad_b200.ops.
Models are held as a training program holds them: parameters, gradients and moments in one flat buffer each, every
tensor a view that starts at a multiple of 256 elements.
"""
import math

import torch

own = False

BLOCK = 256          # elements that share one exponent in the 8-bit moments; also the tensors' alignment in a buffer
MASK = 0xFFFFFFFF
BETA1, BETA2, EPS, DECAY, LR = 0.9, 0.999, 1e-8, 0.1, 3e-4
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases ----
def _decoder(layers, d, kv, ffn, vocab):
    """Tensor sizes of a decoder: the embedding, nine tensors a layer, the last norm, the head."""
    one = [d, d * d, kv * d, kv * d, d * d, d, ffn * d, ffn * d, ffn * d]
    return [vocab * d] + one * layers + [d, vocab * d]


def _sizes(case):
    """The tensors' sizes, from the model's widths or from a text of sizes."""
    if case["model"] == "decoder":
        return _decoder(case["layers"], case["d"], case["kv"], case["ffn"], case["vocab"])
    return [int(s) for s in case["sizes"].split()]


def listed():
    block = dict(model="sizes", sizes=" ".join(map(str, [256, 256] + [65536] * 4 + [256, 256] + [262144] * 3)))
    big = dict(model="decoder", layers=16, d=2048, kv=512, ffn=8192, vocab=32000)
    return [
        # one sequence of 128 tokens in the small fp32 block: a few microseconds, latency alone
        dict(name="norm fwd block", op="norm_fwd", dtype="f32", rows=128, cols=256),
        # a training batch of 16 x 1024 tokens at the decoder's width
        dict(name="norm fwd batch", op="norm_fwd", dtype="bf16", rows=16384, cols=2048),
        # rows whose length is odd, so that they start at any address
        dict(name="norm fwd odd", op="norm_fwd", dtype="bf16", rows=3001, cols=5003),
        dict(name="norm bwd block", op="norm_bwd", dtype="f32", rows=128, cols=256),
        dict(name="norm bwd batch", op="norm_bwd", dtype="bf16", rows=16384, cols=2048),
        # the feed-forward width in fp32: the longest rows in use
        dict(name="norm bwd wide", op="norm_bwd", dtype="f32", rows=2047, cols=8192),
        # clipping: the norm over the small block's gradients, and over the 1.1-billion-parameter decoder's
        dict(name="grad norm block", op="grad_norm", grad="f32", **block),
        dict(name="grad norm decoder", op="grad_norm", grad="bf16", **big),
        # the small block with everything in fp32
        dict(name="adamw block", op="adamw", param="f32", grad="f32", copy=False, **block),
        # mixed precision: fp32 weights, bf16 gradients, and the bf16 copy of the weights that the next pass reads
        dict(name="adamw decoder", op="adamw", param="f32", grad="bf16", copy=True, **big),
        # small and ragged tensors (biases, norms, an odd projection) in bf16 with 8-bit moments
        dict(name="adamw8 ragged", op="adamw8", param="bf16", grad="bf16", copy=False, model="sizes",
             sizes=" ".join(map(str, [1, 255, 257, 2048, 2048, 1000 * 1001, 77 * 513, 2047, 300001]))),
        # the decoder again, its moments in 2 bytes a parameter in place of 8
        dict(name="adamw8 decoder", op="adamw8", param="f32", grad="bf16", copy=True, **big),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "norm_bwd", "grad_norm", "adamw", "adamw8"])
    if op.startswith("norm"):
        cols = _log_int(rng, 32, 16384)
        if rng.random() < 0.5:
            cols = max(32, cols // 8 * 8)
        rows = _log_int(rng, 1, max(1, min(32768, (1 << 25) // cols)))
        return dict(op=op, dtype=rng.choice(["f32", "bf16"]), rows=rows, cols=cols)
    top = 10 ** rng.uniform(3.0, 7.3)
    sizes = [_log_int(rng, 1, int(top)) for _ in range(_log_int(rng, 1, 200))]
    while sum(sizes) > (1 << 28):
        sizes.pop()
    case = dict(op=op, model="sizes", sizes=" ".join(map(str, sizes)), grad=rng.choice(["f32", "bf16"]))
    if op != "grad_norm":
        case["param"] = "f32" if case["grad"] == "f32" else rng.choice(["f32", "bf16"])
        case["copy"] = case["param"] == "f32" and rng.random() < 0.5
    return case


# ----------------------------------------------------------------- inputs ----
def _views(flat, sizes):
    out, at = [], 0
    for n in sizes:
        out.append(flat[at:at + n])
        at += -(-n // BLOCK) * BLOCK
    return out


def _prepare_norm(case, gen):
    M, N, dt = case["rows"], case["cols"], DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    # rows of different size and offset, as a residual stream has them
    x = (rand(M, N) * (0.5 + rand(M, 1).abs()) + 0.5 * rand(M, 1)).to(dt)
    s = dict(case=case, x=x, w=(1 + 0.1 * rand(N)).to(dt), b=(0.1 * rand(N)).to(dt), eps=1e-5)
    if case["op"] == "norm_bwd":
        xf = x.float()
        s["mean"] = xf.mean(1)
        s["rstd"] = torch.rsqrt((xf - s["mean"][:, None]).square().mean(1) + s["eps"])
        s["dy"] = (0.01 * rand(M, N)).to(dt)
    return s


def _prepare_model(case, gen):
    sizes = _sizes(case)
    nb = torch.tensor([-(-n // BLOCK) for n in sizes])
    total = int(nb.sum()) * BLOCK
    real = torch.zeros(total, dtype=torch.bool, device="cuda")
    for part in _views(real, sizes):
        part.fill_(True)
    # one size of gradient for each block of elements, over two decades
    width = (10.0 ** (torch.rand(total // BLOCK, 1, device="cuda", generator=gen) * 2 - 4))

    def rand(scale):
        r = torch.randn(total // BLOCK, BLOCK, device="cuda", generator=gen).mul_(scale).view(-1)
        return r.mul_(real)

    s = dict(case=case, sizes=sizes, g=rand(width).to(DTYPES[case["grad"]]))
    s["grads"] = _views(s["g"], sizes)
    if case["op"] == "grad_norm":
        return s
    s["p"] = rand(0.02).to(DTYPES[case["param"]])
    s["params"] = _views(s["p"], sizes)
    s["copy"] = s["p"].bfloat16() if case["copy"] else None
    s["copies"] = _views(s["copy"], sizes) if case["copy"] else None
    s["step"] = 100
    s["scale"] = 0.5 + torch.rand(1, device="cuda", generator=gen)   # what clipping leaves of the gradients
    m = rand(0.3 * width)
    v = rand(width).square_().mul_(0.5).add_(width.square().expand(-1, BLOCK).reshape(-1) * 0.3).mul_(real)
    if case["op"] == "adamw":
        s["m"], s["v"] = m, v
        s["ms"], s["vs"] = _views(m, sizes), _views(v, sizes)
        return s
    s["seed"] = 12345
    for name, x in (("m", m), ("s", v.sqrt_())):
        x = x.view(-1, BLOCK)
        e = (torch.frexp(x.abs().amax(1))[1] + 119).clamp(0, 247)
        s[name] = torch.ldexp(x, (127 - e)[:, None].float()).to(torch.float8_e4m3fn).view(-1)
        s[name + "_exp"] = e.to(torch.uint8)
        s[name + "s"] = _views(s[name], sizes)
        s[name + "_exps"] = list(s[name + "_exp"].split(nb.tolist()))
    # where each block lies: its tensor's number, and its own within the tensor
    s["tensor"] = torch.repeat_interleave(torch.arange(len(sizes)), nb).cuda()
    first = torch.cumsum(nb, 0) - nb
    s["block"] = torch.arange(total // BLOCK, device="cuda") - first.cuda()[s["tensor"]]
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = (_prepare_norm if case["op"].startswith("norm") else _prepare_model)(case, gen)
    if own and case["op"].startswith("adamw"):   # the optimiser that the program keeps
        from teenygrad_b200 import ops

        state = dict(m=s["ms"], v=s["vs"]) if case["op"] == "adamw" else dict(
            m=s["ms"], m_exp=s["m_exps"], s=s["ss"], s_exp=s["s_exps"])
        s["plan"] = ops.AdamW(s["params"], s["grads"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                              copies=s["copies"], state_bits=32 if case["op"] == "adamw" else 8, seed=s.get("seed", 0),
                              state=state, step_count=s["step"])
    return s


# ------------------------------------------------------------ plain forms ----
def _norm_fwd(s):
    x = s["x"].float()
    mean = x.sum(1) / x.shape[1]
    d = x - mean[:, None]
    rstd = 1 / torch.sqrt((d * d).sum(1) / x.shape[1] + s["eps"])
    y = d * rstd[:, None] * s["w"].float() + s["b"].float()
    return y.to(s["x"].dtype), mean, rstd


def _norm_bwd(s):
    dy, x, N = s["dy"].float(), s["x"].float(), s["x"].shape[1]
    rstd = s["rstd"][:, None]
    xhat = (x - s["mean"][:, None]) * rstd
    a = dy * s["w"].float()
    c1 = a.sum(1, keepdim=True) / N
    c2 = (a * xhat).sum(1, keepdim=True) / N
    dx = rstd * (a - c1 - xhat * c2)
    return dx.to(s["x"].dtype), (dy * xhat).sum(0), dy.sum(0)


def _grad_norm(s):
    g = s["g"].float()
    norm = torch.sqrt((g * g).sum(dtype=torch.float64))
    scale = torch.clamp(1.0 / (norm + 1e-6), max=1.0)
    return norm.float().reshape(1), scale.float().reshape(1)


def _apply(s, m, root):
    """The parameters' step from the first moment and the second's root."""
    t = s["step"]
    p = s["p"].float()
    step = m / (root / math.sqrt(1 - BETA2 ** t) + EPS)
    p = p * (1 - LR * DECAY) - step * (LR / (1 - BETA1 ** t))
    s["p"].copy_(p)
    if s["copy"] is not None:
        s["copy"].copy_(p)


def _adamw(s):
    s["step"] += 1
    g = s["g"].float() * s["scale"]
    s["m"].copy_(s["m"] * BETA1 + g * (1 - BETA1))
    s["v"].copy_(s["v"] * BETA2 + g * g * (1 - BETA2))
    _apply(s, s["m"], torch.sqrt(s["v"]))
    return {k: s[k] for k in ("p", "copy", "m", "v")}


def _mix(x):
    """Mixes 32-bit words held in 64 (a bijection on them)."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & MASK
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & MASK
    return x ^ (x >> 16)


def _bits(s):
    """32 random bits for each element, a function of the seed, the step, the tensor and the place in it."""
    key = _mix(_mix(_mix(torch.full_like(s["tensor"], s["seed"]) & MASK) ^ (s["step"] & MASK)) ^ s["tensor"])
    place = s["block"][:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    key = key[:, None] + (place >> 32) * 0xBB67AE85
    return _mix((key + (place & MASK) * 0x9E3779B1) & MASK)


def _power(e):
    """2 ** (e - 127) in 32 bits, exactly, the subnormal one among them."""
    return torch.where(e == 0, torch.full_like(e, 0x00400000), e << 23).view(torch.float32)


def _decode(code, exp):
    return code.float().view(-1, BLOCK) * _power(exp.int())[:, None]


def _encode(x, u, keep):
    """Blocks of 32-bit values to 8-bit codes and an exponent a block. `u`: 16 random bits an element, which round
    to the code above with the probability of the rest. `keep`: what is above zero stays above it."""
    size = x.abs()
    fine = torch.isfinite(size)
    top = torch.where(fine, size, 0.0).amax(1)
    e = ((top.view(torch.int32) >> 23) - 7).clamp(min=0)
    y = size * _power(254 - e)[:, None]
    low = y < 2.0 ** -6
    y = torch.where(low, y + 2.0 ** -6, y)
    code = ((y.view(torch.int32) + (u << 4 | 8).int()) >> 20) - torch.where(low, 968, 960)
    if keep:
        code = torch.where((size > 0) & (code == 0), 1, code)
    code = torch.where(fine, torch.where((x < 0) & (code > 0), code | 0x80, code), 0x7F)
    return code.to(torch.uint8).view(-1).view(torch.float8_e4m3fn), e.to(torch.uint8)


def _adamw8(s):
    s["step"] += 1
    g = s["g"].float().view(-1, BLOCK) * s["scale"]
    old = _decode(s["s"], s["s_exp"])
    root = torch.sqrt(old * old * BETA2 + g * g * (1 - BETA2))
    m = _decode(s["m"], s["m_exp"]) * BETA1 + g * (1 - BETA1)
    _apply(s, m.view(-1), root.view(-1))
    bits = _bits(s)
    for name, x, u in (("m", m, bits & 0xFFFF), ("s", root, bits >> 16)):
        code, e = _encode(x, u, name == "s")
        s[name].view(torch.uint8).copy_(code.view(torch.uint8))
        s[name + "_exp"].copy_(e)
    return {k: s[k] for k in ("p", "copy", "m", "m_exp", "s", "s_exp")}


# ------------------------------------------------------------------- run ----
def run(s):
    op = s["case"]["op"]
    if not own:
        return dict(norm_fwd=_norm_fwd, norm_bwd=_norm_bwd, grad_norm=_grad_norm, adamw=_adamw, adamw8=_adamw8)[op](s)
    from teenygrad_b200 import ops

    if op == "norm_fwd":
        return ops.layer_norm(s["x"], s["w"], s["b"], s["eps"], return_stats=True)
    if op == "norm_bwd":
        return ops.layer_norm_backward(s["dy"], s["x"], s["w"], s["mean"], s["rstd"])
    if op == "grad_norm":
        return ops.grad_norm(s["grads"], max_norm=1.0)
    s["plan"].step(grad_scale=s["scale"])
    return {k: s[k] for k in (("p", "copy", "m", "v") if op == "adamw" else ("p", "copy", "m", "m_exp", "s", "s_exp"))}


def work(case):
    op = case["op"]
    if op.startswith("norm"):
        M, N, e = case["rows"], case["cols"], 4 if case["dtype"] == "f32" else 2
        if op == "norm_fwd":   # x in, y out, weight and bias in, two numbers a row out
            return dict(bytes=2 * M * N * e + 2 * N * e + 8 * M, flops=7 * M * N)
        return dict(bytes=3 * M * N * e + N * e + 8 * M + 8 * N, flops=14 * M * N)
    n, nb = sum(_sizes(case)), sum(-(-k // BLOCK) for k in _sizes(case))
    g = 4 if case["grad"] == "f32" else 2
    if op == "grad_norm":
        return dict(bytes=n * g + 8, flops=2 * n)
    p = (8 if case["param"] == "f32" else 4) + (2 if case["copy"] else 0)
    if op == "adamw":
        return dict(bytes=n * (p + g + 16), flops=16 * n)
    return dict(bytes=n * (p + g + 4) + 4 * nb, flops=40 * n)


# ----------------------------------------------------------------- exact ----
def _exact_code(x, u, keep):
    """_encode's definition in 64 bits: the grid of a block is that of its largest value's binade."""
    size = x.abs()
    top = torch.frexp(size.amax(1, keepdim=True))[1]         # largest = f * 2 ** top, f in [1/2, 1)
    e = (top - 8).clamp(min=-127)
    y = size * torch.pow(2.0, -e.double())
    step = torch.pow(2.0, (torch.frexp(y)[1].clamp(min=-5) - 4).double())
    code = torch.floor(y / step + (u.double() + 0.5) / 65536) * step
    if keep:
        code = torch.where((size > 0) & (code == 0), 2.0 ** -9, code)
    return (torch.sign(x) * code).view(-1)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "norm_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        rstd = (var + s["eps"]).rsqrt()
        return torch.addcmul(s["b"].double(), (x - mean) * rstd, s["w"].double()), mean.view(-1), rstd.view(-1)
    if op == "norm_bwd":
        # the gradient of sum(dy * norm(x)), by automatic differentiation
        x, w = s["x"].double().requires_grad_(), s["w"].double().requires_grad_()
        b = torch.zeros_like(w).requires_grad_()
        y = torch.nn.functional.layer_norm(x, (x.shape[1],), w, b, s["eps"])
        return torch.autograd.grad(y, (x, w, b), s["dy"].double())
    if op == "grad_norm":
        norm = sum(float(g.double().square().sum()) for g in s["grads"]) ** 0.5
        return (torch.tensor([norm], dtype=torch.float64), torch.tensor([min(1.0, 1.0 / (norm + 1e-6))], dtype=torch.float64))
    t = s["step"] = s["step"] + 1
    g = s["g"].double() * s["scale"].double()
    if op == "adamw":
        m, v = torch.lerp(g, s["m"].double(), BETA1), torch.lerp(g.square_(), s["v"].double(), BETA2)
        out = dict(m=m, v=v)
        root = v.sqrt()
    else:
        def held(name):
            e = s[name + "_exp"].double() - 127
            return (s[name].double().view(-1, BLOCK) * torch.pow(2.0, e)[:, None]).view(-1)

        m, root = torch.lerp(g, held("m"), BETA1), torch.lerp(g.square(), held("s").square_(), BETA2).sqrt_()
        del g
        bits = _bits(s)
        out = dict(m=_exact_code(m.view(-1, BLOCK), bits & 0xFFFF, False), m_exp=None,
                   s=_exact_code(root.view(-1, BLOCK), bits >> 16, True), s_exp=None)
        del bits
    p = s["p"].double()
    out["p"] = p - LR * (m / (1 - BETA1 ** t) / (root / (1 - BETA2 ** t) ** 0.5 + EPS) + DECAY * p)
    out["copy"] = out["p"] if s["copy"] is not None else None
    return out
