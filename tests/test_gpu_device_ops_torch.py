"""The device-pointer operators among torch's own work: streams, captured graphs, autograd's view of their outputs."""
import pytest
from test_gpu_device_ops import dev, dtype_of, here, i32, packed_space, randn, shared_space, torch_  # noqa: F401

pytestmark = pytest.mark.gpu


def calls(dev):
    """(name, inputs to fill, outputs, call) of each operator on small buffers."""
    torch = torch_()
    dt = dtype_of("bf16")
    q, k, v = randn(1, 30, 8, 128, dtype=dt), randn(2, 900, 1, 128, dtype=dt), randn(3, 900, 1, 128, dtype=dt)
    off, ko = i32([0, 30]), i32([0, 900])
    out, lse = torch.zeros_like(q), torch.zeros(30, 8, device="cuda")
    space = packed_space(dev, q, k, off)
    sq, sk, lens = q[:5], k.view(5, 180, 1, 128), i32([1, 0, 180, 33, 70])
    sout, slse = torch.zeros_like(sq), torch.zeros(5, 8, device="cuda")
    sspace = shared_space(dev, sq, k, sk)
    x = randn(4, 6, 20000, dtype=torch.float32)
    y, tokens = torch.zeros_like(x), i32([0] * 6)
    hist, hoff, pen = i32(list(range(60))), i32([10 * i for i in range(7)]), torch.full((6,), 1.5, device="cuda")
    return [
        ("packed", q, (out, lse), lambda **kw: dev.attention_packed(q, k, v, off, ko, out, lse=lse, workspace=space, **kw)),
        ("shared", q, (sout, slse),
         lambda **kw: dev.attention_shared(sq, k, v, sk, sk, lens, sout, lse=slse, workspace=sspace, **kw)),
        ("logits", x, (y, tokens), lambda **kw: dev.adjust_logits(x, y, tokens, history=hist, history_offsets=hoff,
                                                                  repetition=pen, **kw)),
    ]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_without_a_stream_a_call_follows_torchs_work_and_precedes_it(dev, which):
    """The input's producer is late, the output's consumer follows at once; both on torch's current stream."""
    torch = torch_()
    _, fill, outs, call = calls(dev)[which]
    fresh = (randn(9, *fill.shape, dtype=torch.float32) * 2).to(fill.dtype)
    fill.copy_(fresh)
    assert call(stream=here())
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    fill.zero_()
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # some 50 ms
        fill.copy_(fresh)
        assert call()
        got = [o.clone() for o in outs]
        for o in outs:
            o.zero_()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    dev.status()
    assert all(not o.any() for o in outs)  # nothing wrote them afterwards


@pytest.mark.parametrize("which", [0, 1, 2])
def test_without_a_stream_a_call_is_part_of_a_captured_graph(dev, which):
    torch = torch_()
    _, fill, outs, call = calls(dev)[which]
    assert call(stream=here())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call()
    fresh = (randn(9, *fill.shape, dtype=torch.float32) * 2).to(fill.dtype)
    fill.copy_(fresh)
    assert call(stream=here())
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    for o in outs:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    dev.status()


def test_a_disposed_backend_is_refused_with_and_without_a_stream(built_lib):
    from funasrnet_b200.backend import CudaFloatBackend
    from funasrnet_b200.device_ops import DeviceOps

    backend = CudaFloatBackend(0)
    ops = DeviceOps(backend)
    _, _, outs, call = calls(ops)[2]
    assert call()
    torch_().cuda.synchronize()
    backend.dispose()
    for o in outs:
        o.fill_(7)
    for kw in ({}, {"stream": here()}):
        with pytest.raises(RuntimeError, match="disposed"):
            call(**kw)
    torch_().cuda.synchronize()
    assert all((o == 7).all() for o in outs)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_call_raises_the_version_of_its_outputs(dev, which):
    """Autograd refuses a backward pass through a tensor that a call has overwritten since it was saved."""
    torch = torch_()
    _, _, outs, call = calls(dev)[which]
    before = [o._version for o in outs]
    assert call(stream=here())
    assert all(o._version > b for o, b in zip(outs, before))
    if which < 2:
        w = torch.ones_like(outs[0], requires_grad=True)
        loss = (w * outs[0]).sum()
        assert call(stream=here())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    torch.cuda.synchronize()


def test_tensors_that_require_grad_are_refused_and_inference_tensors_taken(dev):
    torch = torch_()
    dt = dtype_of("f16")
    q, k = randn(1, 4, 2, 64, dtype=dt), randn(2, 9, 2, 64, dtype=dt)
    off, ko = i32([0, 4]), i32([0, 9])
    out = torch.full_like(q, 7.0)
    leaf = q.clone().requires_grad_()
    for args in ((leaf, k, k), (q, k.clone().requires_grad_(), k), (q, k, k.clone().requires_grad_())):
        with pytest.raises(ValueError, match="requires grad"):
            dev.attention_packed(*args, off, ko, out, stream=here())
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    with torch.no_grad():
        assert dev.attention_packed(leaf, k, k, off, ko, out, stream=here())
    with torch.inference_mode():
        out2 = torch.zeros_like(q)
        assert dev.attention_packed(q, k, k, off, ko, out2, stream=here())
    torch.cuda.synchronize()
    assert torch.equal(out, out2)
    assert dev.attention_packed(q, k, k, off, ko, out2, stream=here())  # an inference tensor outside that mode
    torch.cuda.synchronize()
    assert torch.equal(out, out2)


def test_graphs_of_every_chain_of_kernels_replayed_at_once(dev):
    """Two captured graphs with a workspace each, of the calls that launch several kernels (packed keys cut and joined; the
    prefix on the tensor cores, own keys beside it, join), replayed on two streams at once with other inputs."""
    torch = torch_()
    dt = dtype_of("f16")

    class Chain:
        def __init__(self, seed):
            self.q, self.k, self.v = (randn(seed + i, n, h, 128, dtype=dt) for i, (n, h) in enumerate(((64, 16), (2600, 8), (2600, 8))))
            self.sk, self.sv = (randn(seed + i, 64, 90, 8, 128, dtype=dt) for i in (3, 4))
            self.qo, self.ko = i32([0, 1, 64]), i32([0, 2000, 2600])
            self.lens = i32([(seed + 7 * i) % 91 for i in range(64)])
            self.outs = [torch.zeros_like(self.q), torch.zeros(64, 16, device="cuda"), torch.zeros_like(self.q),
                         torch.zeros(64, 16, device="cuda")]
            self.spaces = [packed_space(dev, self.q, self.k, self.qo), shared_space(dev, self.q, self.k, self.sk)]
            assert all(s.numel() > 16 for s in self.spaces)

        def __call__(self):
            for _ in range(3):  # the second call's kernels follow the first one's in the same workspace
                assert dev.attention_packed(self.q, self.k, self.v, self.qo, self.ko, self.outs[0], lse=self.outs[1],
                                            workspace=self.spaces[0], stream=here())
                assert dev.attention_shared(self.q, self.k, self.v, self.sk, self.sv, self.lens, self.outs[2], lse=self.outs[3],
                                            workspace=self.spaces[1], stream=here())

    chains = [Chain(1), Chain(50)]
    for c in chains:
        c()
    torch.cuda.synchronize()
    graphs = []
    for c in chains:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            c()
    streams = [torch.cuda.Stream() for _ in chains]
    for turn in range(4):
        want = []
        for c in chains:
            c.q.copy_(randn(100 + turn, *c.q.shape, dtype=dt))
            c()
            torch.cuda.synchronize()
            want.append([o.clone() for o in c.outs])
            for o in c.outs:
                o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for c, w in zip(chains, want):
            assert all(torch.equal(a, b) for a, b in zip(c.outs, w)), f"turn {turn}"
    dev.status()
