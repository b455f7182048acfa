"""Host threads that share a device's context: each call of the library finds the stream of the thread that makes it.

A fake of the library stands in for the GPU; it notes the stream that the context has when a call begins and when it ends."""
import ctypes
import threading
import time
import types

import pytest

torch = pytest.importorskip("torch")

from teenygrad_b200 import decoder, dist, graph, ops  # noqa: E402

# calls that ask for sizes or free memory: no stream has a part in them
NO_STREAM = {"tb_workspace_bytes", "tb_output_row_stride", "tb_conv2d_workspace_size", "tb_decoder_destroy", "tb_graph_destroy"}


class FakeLibrary:
    def __init__(self, stream_of):
        self.stream, self.stream_of, self.bad, self.calls = None, stream_of, [], set()

    def tb_set_stream(self, ctx, stream):
        self.stream = getattr(stream, "value", stream)
        return 0

    def __getattr__(self, name):
        def call(*args):
            if name in NO_STREAM:
                return 0
            self.calls.add(name)
            before, mine = self.stream, self.stream_of()
            time.sleep(1e-4)   # as a call without the interpreter's lock: other threads run
            if before != mine or self.stream != mine:
                self.bad.append(name)
            return 0
        return call


def calls():
    """A call of each operator that a CPU tensor reaches the library with."""
    x, w, sq = torch.ones(4, 8), torch.ones(8), torch.ones(8, 8)
    q = torch.ones(8, 8, dtype=torch.int8)
    heads, img, kern = torch.ones(1, 2, 4, 8), torch.ones(1, 2, 5, 5), torch.ones(3, 2, 3, 3)
    ids, rows = torch.zeros(4, dtype=torch.int32), torch.ones(4)
    dec, g, comm = (object.__new__(c) for c in (decoder.Decoder, graph.Graph, dist.Comm))
    for o in (dec, g, comm):
        o.device, o.ctx, o._h = 0, ctypes.c_void_p(1), ctypes.c_void_p(1)
    comm.world = 2
    return [
        lambda: ops.rms_norm(x, w), lambda: ops.layer_norm(x, w, w), lambda: ops.layer_norm(x, w, w, return_stats=True),
        lambda: ops.silu(x), lambda: ops.swiglu(x, x), lambda: ops.add(x, x), lambda: ops.linear(x, sq, w),
        lambda: ops.linear_chain([dict(x=x, w=sq, y=x)]), lambda: ops.linear_padded(x, sq), lambda: ops.matmul(x, sq),
        lambda: ops.quantize_int8(sq), lambda: ops.dequantize_int8(q, w), lambda: ops.int8_linear(x, q, w),
        lambda: ops.attention(heads, heads, heads), lambda: ops.rope(heads[0], ids), lambda: ops.embedding(sq, ids),
        lambda: ops.argmax(x), lambda: ops.bn_fold(w, w, w, w), lambda: ops.batch_norm_inference(x, w, w, w, w),
        lambda: ops.conv2d(img, kern), lambda: ops.conv2d_pack_weights(kern), lambda: ops.rms_norm_backward(x, x, w, rows),
        lambda: ops.layer_norm_backward(x, x, w, rows, rows), lambda: ops.linear_backward(x, sq, x),
        lambda: ops.attention_backward(heads, heads, heads, heads, heads, rows),
        lambda: ops.conv2d_backward(torch.ones(1, 3, 3, 3), img, kern), ops.device_error,
        dec.prepare, dec.seq_len, lambda: dec.init_random(1), lambda: dec.fill_kv_random(ids, 3), g.launch,
        lambda: comm.all_gather(ids),
    ]


@pytest.fixture
def fake(monkeypatch):
    local = threading.local()
    lib = FakeLibrary(lambda: local.stream)
    for m in (ops, decoder, graph, dist):
        monkeypatch.setattr(m, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_ctxs", {0: ctypes.c_void_p(1)})
    monkeypatch.setattr(ops, "_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_same", lambda *ts: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: types.SimpleNamespace(cuda_stream=local.stream))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: local.stream, raising=False)
    lib.local = local
    return lib


def test_every_call_is_made_on_its_threads_stream(fake):
    errors = []

    def work(k):
        fake.local.stream = 100 + k
        try:
            todo = calls()
            for r in range(20):
                for i in range(len(todo)):
                    todo[(i * (k + 1) + r) % len(todo)]()   # in another order in each thread
        except Exception as e:   # pragma: no cover - shown by the assertion
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert not fake.bad, sorted(set(fake.bad))
    assert len(fake.calls) >= 29


def test_a_refused_call_lets_the_others_go_on(fake):
    fake.local.stream = 1
    with pytest.raises(ValueError):
        with ops._on():
            raise ValueError
    done = []

    def work():
        fake.local.stream = 2
        ops.add(torch.ones(3), torch.ones(3))
        done.append(fake.stream)

    t = threading.Thread(target=work)
    t.start()
    t.join(10)
    assert done == [2] and not fake.bad


def test_threads_that_step_one_optimiser_have_their_own_rates(fake, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    opt = object.__new__(ops.AdamW)
    opt.__dict__.update(_handle=ctypes.c_void_p(1), _destroy=lambda h: 0, _hyper=ops._AdamWHyper(), _lists=(), _at=[], device=0,
                        lr=1.0, _step=0, _step_dev=None, _captured=[], params=[], grads=[])
    seen, errors = [], []

    def step(handle, hyper):
        first = (hyper._obj.lr, hyper._obj.step)
        time.sleep(1e-4)
        seen.append((fake.local.stream, *first, hyper._obj.lr))
        return 0

    fake.tb_adamw_step = step

    def work(k):
        fake.local.stream = 100 + k
        try:
            for _ in range(200):
                opt.step(lr=100.0 + k)
        except Exception as e:   # pragma: no cover - shown by the assertion
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert all(stream == lr == later for stream, lr, _, later in seen)
    assert [n for _, _, n, _ in seen] == list(range(1, 601)) and opt.step_count == 600
    opt._handle = None
