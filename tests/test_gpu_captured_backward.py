"""What a captured backward pass is held to, on streams that are not captured: a leaf's other graph was made on another stream, so
its gradient would be accumulated there.  (The forward call is told that it is captured.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _calls():
    """name -> (leaf's shape, call of the host entry)"""
    from came_amd import _lib
    host = _lib.host()
    x, w = torch.randn(3, 5, 16, device="cuda"), torch.randn(24, 16, device="cuda")
    down, t = torch.randn(8, 24, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    silu = 0
    return {
        "gated_ffn": ((24, 16), lambda leaf, s, c: host.gated_ffn(x, leaf, w, down, silu, s, c)),  # its weight
        "gated_ffn x": ((3, 5, 16), lambda leaf, s, c: host.gated_ffn(leaf, w, w, down, silu, s, c)),  # reshaped
        "gated_ffn converted": ((24, 16), lambda leaf, s, c: host.gated_ffn(x.bfloat16(), leaf.bfloat16(), w.bfloat16(), down.bfloat16(), silu, s, c)),
        "embedding of a slice": ((9, 40), lambda leaf, s, c: host.embedding(t, leaf[:, 3:20], 1.0, -1, s, c)),
        "rms_norm reshaped": ((6, 16), lambda leaf, s, c: host.rms_norm(leaf.view(2, 3, 16), w[0], None, 1e-6, s, c)[0]),
        "token_log_probs transposed": ((16, 4), lambda leaf, s, c: host.token_log_probs(leaf.t(), t, 0, s, c)[0]),
    }


@pytest.mark.parametrize("name", ["gated_ffn", "gated_ffn x", "gated_ffn converted", "embedding of a slice", "rms_norm reshaped",
                                  "token_log_probs transposed"])
def test_a_leaf_whose_gradient_lies_on_another_stream(name):
    shape, fn = _calls()[name]
    leaf = torch.randn(shape, device="cuda", requires_grad=True)

    def call(captured):
        return fn(leaf, torch.cuda.current_stream().cuda_stream, captured).sum()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(True).backward()  # no other graph of the leaf
        other = leaf.grad.clone()
    torch.cuda.synchronize()
    alive = leaf * 2  # on the first stream
    with torch.cuda.stream(side):
        y = call(True)
        with pytest.raises(RuntimeError, match=f"{name.split()[0]}.*another stream"):
            y.backward()
        g, = torch.autograd.grad(call(True), leaf)  # accumulates nothing
        call(False).backward()
    torch.cuda.synchronize()
    assert torch.equal(g, other) and torch.equal(leaf.grad, 2 * other) and alive.shape == shape
    del alive, y
    with torch.cuda.stream(side):
        call(True).backward()
    torch.cuda.synchronize()
    assert torch.equal(leaf.grad, 3 * other)


def test_a_leaf_whose_stream_is_captured_too(monkeypatch):
    """A capture of two streams: the leaf's gradient may be accumulated on the other one.  (torch is made to say that it is
    captured.)"""
    for name, (shape, fn) in _calls().items():
        leaf = torch.randn(shape, device="cuda", requires_grad=True)
        first, side = torch.cuda.current_stream(), torch.cuda.Stream()
        alive = leaf * 2
        with monkeypatch.context() as m:
            m.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: torch.cuda.current_stream() == first)
            side.wait_stream(first)
            with torch.cuda.stream(side):
                fn(leaf, side.cuda_stream, True).sum().backward()
        torch.cuda.synchronize()
        got, leaf.grad = leaf.grad, None
        fn(leaf, first.cuda_stream, False).sum().backward()
        assert torch.equal(got, leaf.grad), name
        assert torch.cuda.current_stream() == first and alive.shape == shape


def test_a_block_is_captured_and_replayed():
    """The block's backward pass in a graph, against eager work between the replays."""
    from came_amd import gated_ffn
    gen = torch.Generator().manual_seed(0)
    x, gate, up, down = (torch.randn(*s, generator=gen).cuda().requires_grad_() for s in ((2, 40, 64), (96, 64), (96, 64), (64, 96)))

    def step():
        for p in (x, gate, up, down):
            p.grad = None
        y = gated_ffn(x, gate, up, down)
        y.square().sum().backward()
        return [y.detach(), x.grad, gate.grad, up.grad, down.grad]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(2, 40, 64, generator=gen).cuda())
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in held]
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, kept))
