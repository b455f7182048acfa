"""Host threads with streams of their own: operators of every kind side by side, each read on its thread's stream."""
import threading

import pytest

from gpu_util import dev, torch

pytestmark = pytest.mark.gpu


def test_operators_of_all_kinds_in_threads():
    dev()
    from teenygrad_b200 import ops as o
    from teenygrad_b200.decoder import Decoder, DecoderConfig
    K = 3

    def made(k):
        g = torch.Generator(device="cuda").manual_seed(k)

        def rand(*s):
            return torch.randn(*s, device="cuda", generator=g)

        return dict(x=rand(300, 256), w=rand(128, 256), dy=rand(300, 128), gamma=rand(256), img=rand(2, 64, 9, 9).bfloat16(),
                    kern=rand(64, 64, 3, 3).bfloat16(), p=[rand(5000), rand(77)], g=[rand(5000), rand(77)])

    def work(t, opt):
        y, mean, rstd = o.layer_norm(t["x"], t["gamma"], t["gamma"], return_stats=True)
        out = [y, mean, rstd, *o.layer_norm_backward(t["x"], t["x"], t["gamma"], mean, rstd)]
        out += [o.linear(t["x"], t["w"]), *o.linear_backward(t["x"], t["w"], t["dy"])]
        out += [o.layer_norm(t["x"], t["gamma"], t["gamma"]), o.silu(t["x"]), o.conv2d(t["img"], t["kern"], pad=1)]
        norm, scale = o.grad_norm(t["g"], max_norm=1.0)
        opt.step(grad_scale=scale)
        return out + [norm, scale] + [p.clone() for p in t["p"]]

    decoder = Decoder(DecoderConfig(n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn_hidden=512, vocab=1000,
                                    max_batch=2, max_seq=64))
    decoder.init_random(seed=1)
    prompt = torch.arange(16, device="cuda", dtype=torch.int32).view(2, 8)
    tokens = decoder.generate(prompt, 4)
    rounds = 30
    data = [made(k) for k in range(K)]
    copies = [made(k) for k in range(K)]
    opts = [o.AdamW(t["p"], t["g"], state_bits=8 if k else 32) for k, t in enumerate(data)]
    refs = [o.AdamW(t["p"], t["g"], state_bits=8 if k else 32) for k, t in enumerate(copies)]
    want = [[work(t, opt) for _ in range(rounds)] for t, opt in zip(copies, refs)]
    torch.cuda.synchronize()
    streams, bad = [torch.cuda.Stream() for _ in range(K + 1)], []

    def run(k):
        try:
            with torch.cuda.stream(streams[k]):
                for r in range(rounds):
                    if k == K:   # its launches are of the programmatic kind
                        if not torch.equal(decoder.generate(prompt, 4), tokens):
                            bad.append("decoder")
                        continue
                    got = work(data[k], opts[k])
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k][r])):
                        bad.append((k, r))
        except Exception as e:   # pragma: no cover - shown by the assertion
            bad.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(K + 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad
