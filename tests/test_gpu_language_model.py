"""The operators around the gated feed-forward block together, as a program trains and serves a model with them."""
import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _reference(model, tokens, bonus, padding):
    """The loss and every gradient in 64 bits, in elementary operations."""
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in model.named_parameters()}
    t, follow = tokens[:, :-1].cpu(), tokens[:, 1:].cpu()
    table = torch.where(torch.arange(p["table"].shape[0])[:, None] == padding, p["table"].detach(), p["table"])

    def norm(h, w):
        return h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w

    h = table[t] * math.sqrt(p["table"].shape[1])
    for k in range(len(model.blocks)):
        y = norm(h, p[f"norms.{k}"])
        g, u = y @ p[f"blocks.{k}.gate"].t(), y @ p[f"blocks.{k}.up"].t()
        h = h + (g * torch.sigmoid(g) * u) @ p[f"blocks.{k}.down"].t()
    logp = torch.log_softmax(norm(h, p[f"norms.{len(model.blocks)}"]) @ p["head"].t(), -1)
    given = follow != padding
    lp = logp.gather(-1, follow[..., None]).squeeze(-1)
    entropy = -(logp.exp() * logp).sum(-1)
    loss = -torch.where(given, lp, 0.0).sum() / given.sum() - bonus * entropy.mean()
    return loss, dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


def test_gradients_of_a_model():
    """Every parameter's gradient in float32.  A product or sum of n <= 1024 terms is off by n 2^-24 of its terms' magnitudes,
    6e-5, which is 32 times as much of a result whose terms have random signs; a dozen operators one after another: 2e-2 at most,
    of the gradient's 2-norm, and as its roundings are random too a tenth of that."""
    import train_language_model as ex
    gen = torch.Generator().manual_seed(1)
    model = ex.Model(301, 96, 200, 3, torch.float32, gen)
    with torch.no_grad():
        for n in model.norms:
            n.copy_(1 + 0.2 * torch.randn(96, generator=gen).cuda())
    tokens = torch.randint(0, 301, (7, 33), generator=gen)
    tokens[3, 20:] = ex.PADDING
    tokens = tokens.cuda()
    loss = ex.loss_of(model(tokens[:, :-1]), tokens[:, 1:], bonus=0.1)
    loss.backward()
    want, grads = _reference(model, tokens, 0.1, ex.PADDING)
    want = float(want.detach())
    assert abs(float(loss.detach()) - want) <= 1e-4 * abs(want)
    for name, p in model.named_parameters():
        g = grads[name]
        assert (p.grad.cpu().double() - g).norm() <= 2e-3 * g.norm(), name
    assert not model.table.grad[ex.PADDING].any()


@pytest.mark.parametrize("name,dtype", [("adamw", "fp32"), ("adamw8bit", "bf16"), ("came8bit", "bf16")])
def test_a_model_is_trained_and_served(name, dtype):
    """The example runs, and the 8-bit head's log probabilities are as near to the trained head's as half a code of each
    operand allows."""
    import train_language_model as ex
    model, losses, unseen = ex.train(12, vocab=500, dim=128, hidden=352, batch=6, length=40, name=name, dtype=dtype, log=lambda *_: None)
    assert len(losses) == 3 and all(math.isfinite(v) for v in losses)
    assert all(torch.isfinite(p).all() for p in model.parameters())
    scorer = ex.Scorer(model)
    r = scorer(unseen, top=4)
    import came_amd
    with torch.no_grad():
        x, h = model.stream(unseen[:, :-1])
        y = came_amd.rms_norm(x.float(), model.norms[-1].float(), residual=h.float())[0].double()
        q, s, _ = came_amd.rms_norm_int8(x, model.norms[-1], residual=h)
        held, head = scorer.head.double() * scorer.scale.double()[:, None], model.head.double()
        logits = y @ head.t()
        # y as codes: half a code, and where h is rounded to its type (rms_norm_int8 takes the rounded one) that rounding, 2^-8 of h
        h_rounding = 0.0 if dtype == "fp32" else 2.0**-8
        ey = 0.5 * s.double()[..., None] + 2 * h_rounding * (y.abs() + y.square().mean(-1, keepdim=True).sqrt())
        off = ey @ held.abs().t() + y.abs() @ (0.5 * scorer.scale.double()[:, None].expand_as(head)).t() + 1e-4
        logp = torch.log_softmax(logits, -1)
        want = logp.gather(-1, unseen[:, 1:, None]).squeeze(-1)
        assert ((r.log_probs.double() - want).abs() <= 2 * off.amax(-1)).all()
        exact = came_amd.int8_linear(q, s, scorer.head, scorer.scale, dtype=torch.float32)
        assert torch.equal(r.top_tokens, torch.sort(exact, dim=-1, descending=True, stable=True).indices[..., :4])


def test_a_step_is_captured_and_replayed():
    """Forward and backward of the whole model in a graph, after a warm-up on its stream, with eager work between replays."""
    import train_language_model as ex
    gen = torch.Generator().manual_seed(2)
    model = ex.Model(200, 64, 96, 2, torch.bfloat16, gen)
    tokens = torch.randint(0, 200, (4, 17), generator=gen).cuda()

    def step():
        for p in model.parameters():
            p.grad = None
        loss = ex.loss_of(model(tokens[:, :-1]), tokens[:, 1:], bonus=0.01)
        loss.backward()
        return [loss.detach(), *(p.grad for p in model.parameters())]

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
        tokens.copy_(torch.randint(0, 200, (4, 17), generator=gen).cuda())
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in held]
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.synchronize()
        assert all(torch.allclose(a.float(), b.float(), rtol=2.0**-7, atol=1e-6) for a, b in zip(eager, kept))


@pytest.mark.parametrize("op", ["embedding", "rms_norm", "token_log_probs"])
def test_a_leaf_whose_gradient_lies_on_another_stream(op):
    """What a captured backward pass is held to, on streams that are not captured: the leaf's other graph was made on another
    stream, so its gradient is accumulated there.  (The forward call is told that it is captured.)"""
    import came_amd
    from came_amd import _lib
    leaf = torch.randn(40, 32, device="cuda", requires_grad=True)
    t = torch.zeros(40, dtype=torch.long, device="cuda")
    w = torch.ones(32, device="cuda")

    def call(captured):
        stream = torch.cuda.current_stream().cuda_stream
        host = _lib.host()
        if op == "embedding":
            return host.embedding(t, leaf, 1.0, -1, stream, captured)
        if op == "rms_norm":
            return host.rms_norm(leaf, w, None, 1e-6, stream, captured)[0]
        return host.token_log_probs(leaf, t, 0, stream, captured)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(True).sum().backward()  # no other graph of the leaf
        other = leaf.grad.clone()
    torch.cuda.synchronize()
    alive = came_amd.embedding(t, leaf)  # on the first stream
    with torch.cuda.stream(side):
        y = call(True)
        with pytest.raises(RuntimeError, match=f"{op}.*another stream"):
            y.sum().backward()
        g, = torch.autograd.grad(call(True).sum(), leaf)  # accumulates nothing
        call(False).sum().backward()
    torch.cuda.synchronize()
    assert torch.equal(g, other) and torch.equal(leaf.grad, 2 * other) and alive.shape == (40, 32)
    del alive, y
    with torch.cuda.stream(side):
        call(True).sum().backward()
    torch.cuda.synchronize()
    assert torch.equal(leaf.grad, 3 * other)


def test_saved_tensors_that_are_made_again():
    """Checkpointed, the operators' saved tensors are thrown away and the forward pass is run again: the same bits."""
    from torch.utils.checkpoint import checkpoint

    from came_amd import embedding, rms_norm, token_log_probs
    gen = torch.Generator().manual_seed(9)
    table, w, head = (torch.randn(*s, generator=gen).cuda().requires_grad_() for s in ((50, 24), (24,), (50, 24)))
    tokens = torch.randint(0, 50, (40,), generator=gen).cuda()

    def loss(table, w, head):
        h = embedding(tokens[:-1], table)
        y, h = rms_norm(h, w, residual=h)
        out = token_log_probs((y + h) @ head.t(), tokens[1:])
        return out.log_probs.sum() + out.entropy.sum()

    want = torch.autograd.grad(loss(table, w, head), (table, w, head))
    got = torch.autograd.grad(checkpoint(loss, table, w, head, use_reentrant=False), (table, w, head))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_tensors_that_are_written():
    """A backward pass whose saved tensors were written after the forward pass raises."""
    from came_amd import embedding, rms_norm, token_log_probs
    w, x = torch.ones(16, device="cuda", requires_grad=True), torch.randn(3, 16, device="cuda", requires_grad=True)
    table, tokens = torch.randn(9, 16, device="cuda", requires_grad=True), torch.zeros(3, dtype=torch.int64, device="cuda")
    y, h = rms_norm(x, w, residual=x)
    h += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = embedding(tokens, table)
    tokens += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    z = x * 1.0
    out = token_log_probs(z, tokens)
    z *= 2
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.log_probs.sum().backward()


def test_calls_of_threads_on_streams_of_their_own():
    """Calls that run at once share nothing."""
    from concurrent.futures import ThreadPoolExecutor

    from came_amd import int8_linear, quantize_rows, rms_norm_int8, token_log_probs
    gen = torch.Generator().manual_seed(4)
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    rows = [torch.randn(t, 512, generator=gen).bfloat16().cuda() for t in (1, 3, 40, 200)]
    weights = quantize_rows(torch.randn(9000, 512, generator=gen).bfloat16().cuda())
    tokens = [torch.randint(0, 9000, (len(x),), generator=gen).cuda() for x in rows]

    def serve(k):
        with torch.no_grad():
            logits = int8_linear(*rms_norm_int8(rows[k], w), *weights)
            return token_log_probs(logits, tokens[k], top=5)

    def in_thread(k):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            out = [serve(k) for _ in range(20)]
        stream.synchronize()
        return out

    want = [serve(k) for k in range(4)]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(4) as pool:
        got = list(pool.map(in_thread, range(4)))
    for k in range(4):
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))
