"""What the embedding, the norm, the 8-bit product and the token log probabilities refuse on the host, and the oracle's gradients
against automatic differentiation."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import came_amd
from came_amd import _lib as L
from oracle import lm_oracle as orc

P = 0x1000  # an aligned address that nothing reads: what is refused launches nothing
BIG = 1 << 50


def _size(name, desc):
    size = ctypes.c_size_t(0)
    rc = getattr(L.load(), f"came8_{name}_workspace_size")(ctypes.byref(desc), ctypes.byref(size))
    return rc, size.value


def _desc(cls, base, **kw):
    d = cls(*base)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


EMBED = (4, 10, 8, 8, -1, 1.0, L.CAME8_BF16, 8, 0)
NORM = (4, 8, 8, 8, 1e-6, L.CAME8_BF16, 0)
INT8 = (100, 8, 16, 16, 16, L.CAME8_BF16, 0)
PROBS = (4, 100, 100, L.CAME8_BF16, 8, 5, 0)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(token_bytes=2), "token_bytes"), (dict(tokens=-1), "tokens"),
    (dict(tokens=1 << 31), "tokens"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 26) + 1), "vocab"), (dict(dim=0, ld_weight=0), "dim"),
    (dict(dim=(1 << 23) + 1, ld_weight=1 << 24), "dim"), (dict(ld_weight=7), "stride"), (dict(ld_weight=(1 << 31) + 1), "stride"),
    (dict(padding=-2), "padding"), (dict(padding=10), "padding")])
def test_embedding_entries_refuse(kw, match):
    lib, e = L.load(), _desc(L.Came8Embedding, EMBED, **kw)
    assert _size("embedding", e)[0] == L.CAME8_EINVAL
    assert lib.came8_embedding_forward(ctypes.byref(e), P, P, P, None) == L.CAME8_EINVAL
    with pytest.raises(RuntimeError, match=match):
        L.check(lib.came8_embedding_backward(ctypes.byref(e), P, P, P, P, BIG, None), "backward")


def test_embedding_entries_refuse_pointers_and_workspaces():
    lib, e = L.load(), _desc(L.Came8Embedding, EMBED)
    need = _size("embedding", e)[1]
    assert need > 0 and lib.came8_embedding_workspace_size(None, None) == L.CAME8_EINVAL
    assert lib.came8_embedding_workspace_size(ctypes.byref(e), None) == L.CAME8_EINVAL
    for i in range(3):
        for bad in (None, P + 1):
            p = [P] * 3
            p[i] = bad
            assert lib.came8_embedding_forward(ctypes.byref(e), *p, None) == L.CAME8_EINVAL
            assert lib.came8_embedding_backward(ctypes.byref(e), *p, P, need, None) == L.CAME8_EINVAL
    assert lib.came8_embedding_forward(ctypes.byref(e), P + 4, P, P, None) == L.CAME8_EINVAL  # of 8-byte tokens
    for ws, n in ((None, need), (P + 8, need), (P, need - 1)):
        assert lib.came8_embedding_backward(ctypes.byref(e), P, P, P, ws, n, None) == L.CAME8_ESPACE
    none = _desc(L.Came8Embedding, EMBED, tokens=0)
    assert lib.came8_embedding_forward(ctypes.byref(none), None, None, None, None) == L.CAME8_OK
    assert lib.came8_embedding_backward(ctypes.byref(none), P, P, P, P, BIG, None) == L.CAME8_EINVAL


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(dim=0), "dim"),
    (dict(dim=(1 << 30) + 1, ld_x=1 << 31, ld_residual=1 << 31), "dim"), (dict(ld_x=7), "stride"), (dict(ld_x=(1 << 31) + 1), "stride"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(ld_residual=7), "stride")])
def test_norm_entries_refuse(kw, match):
    lib, n = L.load(), _desc(L.Came8RmsNorm, NORM, **kw)
    calls = [lib.came8_rms_norm_forward(ctypes.byref(n), P, P, P, P, P, None),
             lib.came8_rms_norm_int8(ctypes.byref(n), P, P, P, P, 16, P, P, None)]
    if match != "eps" and "ld_residual" not in kw:
        calls += [lib.came8_quantize_rows(ctypes.byref(n), P, P, 16, P, None), _size("rms_norm", n)[0]]
    if "ld_residual" not in kw:
        calls.append(lib.came8_rms_norm_backward(ctypes.byref(n), P, P, P, P, P, P, P, BIG, None))
        with pytest.raises(RuntimeError, match=match):
            L.check(calls[-1], "backward")
    assert calls == [L.CAME8_EINVAL] * len(calls)


def test_norm_entries_refuse_pointers_and_workspaces():
    lib, n = L.load(), _desc(L.Came8RmsNorm, NORM)
    need = _size("rms_norm", n)[1]
    ref = ctypes.byref(n)
    for i in range(5):  # x, residual, weight, y, h
        for bad in (None, P + 1):
            p = [P] * 5
            p[i] = bad
            assert lib.came8_rms_norm_forward(ref, *p, None) == L.CAME8_EINVAL
            if i != 3:
                assert lib.came8_rms_norm_int8(ref, *p[:3], P, 16, P, p[4], None) == L.CAME8_EINVAL
    for q, ld, scale in ((None, 16, P), (P + 8, 16, P), (P, 8, P), (P, 24, P), (P, 0, P), (P, 16, None), (P, 16, P + 2)):
        assert lib.came8_rms_norm_int8(ref, P, None, P, q, ld, scale, None, None) == L.CAME8_EINVAL
        assert lib.came8_quantize_rows(ref, P, q, ld, scale, None) == L.CAME8_EINVAL
    assert lib.came8_quantize_rows(ref, None, P, 16, P, None) == L.CAME8_EINVAL
    for i in range(6):  # h, weight, dy, dh, dx, dweight
        p = [P] * 6
        p[i] = P + 1
        assert lib.came8_rms_norm_backward(ref, *p, P, need, None) == L.CAME8_EINVAL
    for ws, size in ((None, need), (P + 8, need), (P, need - 1)):
        assert lib.came8_rms_norm_backward(ref, P, P, P, None, None, P, ws, size, None) == L.CAME8_ESPACE
    assert lib.came8_rms_norm_backward(ref, P, P, P, None, None, None, None, 0, None) == L.CAME8_OK  # nothing is wanted
    none = _desc(L.Came8RmsNorm, NORM, rows=0)
    assert lib.came8_rms_norm_forward(ctypes.byref(none), None, None, None, None, None, None) == L.CAME8_OK
    assert lib.came8_rms_norm_int8(ctypes.byref(none), None, None, None, None, 0, None, None, None) == L.CAME8_OK
    assert lib.came8_quantize_rows(ctypes.byref(none), None, None, 0, None, None) == L.CAME8_OK
    assert lib.came8_rms_norm_backward(ctypes.byref(none), P, P, P, P, P, P, P, BIG, None) == L.CAME8_EINVAL
    assert lib.came8_rms_norm_forward(None, P, P, P, P, P, None) == L.CAME8_EINVAL


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(rows=(1 << 24) + 1), "rows"), ({"in": 0}, "in "), ({"in": 131072}, "131071"),
    (dict(out=0), "out"), (dict(out=(1 << 24) + 1), "out"), (dict(ld_q=7), "stride"), (dict(ld_w=7), "stride"),
    (dict(ld_q=(1 << 20) + 1), "stride"), (dict(rows=1 << 24, out=1 << 13), "2\\^36")])
def test_product_entries_refuse(kw, match):
    lib, l = L.load(), _desc(L.Came8Int8Linear, INT8, **kw)
    assert _size("int8_linear", l)[0] == L.CAME8_EINVAL
    with pytest.raises(RuntimeError, match=match):
        L.check(lib.came8_int8_linear_forward(ctypes.byref(l), P, P, P, P, P, P, P, BIG, None), "forward")


def test_product_entries_refuse_pointers_and_workspaces():
    lib, l = L.load(), _desc(L.Came8Int8Linear, INT8)
    need = _size("int8_linear", l)[1]
    for i in range(6):  # q, scale, w, w_scale, bias, y
        for bad in (None, P + 1):
            if i == 4 and bad is None:  # no bias
                continue
            p = [P] * 6
            p[i] = bad
            assert lib.came8_int8_linear_forward(ctypes.byref(l), *p, P, need, None) == L.CAME8_EINVAL
    l = _desc(L.Came8Int8Linear, INT8, ld_q=1001)  # copied
    need = _size("int8_linear", l)[1]
    assert need >= l.rows * getattr(l, "in")
    for ws, size in ((None, need), (P + 8, need), (P, need - 1)):
        assert lib.came8_int8_linear_forward(ctypes.byref(l), P, P, P, P, None, P, ws, size, None) == L.CAME8_ESPACE
    none = _desc(L.Came8Int8Linear, INT8, rows=0)
    assert lib.came8_int8_linear_forward(ctypes.byref(none), None, None, None, None, None, None, None, 0, None) == L.CAME8_OK


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(token_bytes=1), "token_bytes"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"),
    (dict(vocab=0), "vocab"), (dict(vocab=(1 << 20) + 1, ld=1 << 21), "vocab"), (dict(ld=99), "stride"), (dict(ld=(1 << 31) + 1), "stride"),
    (dict(top=-1), "top"), (dict(top=65), "top"), (dict(vocab=4, ld=4), "top")])
def test_log_prob_entries_refuse(kw, match):
    lib, p = L.load(), _desc(L.Came8LogProbs, PROBS, **kw)
    assert _size("log_probs", p)[0] == L.CAME8_EINVAL
    assert lib.came8_log_probs_backward(ctypes.byref(p), P, P, P, P, P, P, P, None) == L.CAME8_EINVAL
    with pytest.raises(RuntimeError, match=match):
        L.check(lib.came8_log_probs_forward(ctypes.byref(p), P, P, P, P, P, P, P, P, BIG, None), "forward")


def test_log_prob_entries_refuse_pointers_and_workspaces():
    lib, p = L.load(), _desc(L.Came8LogProbs, PROBS, vocab=50000, ld=50000)  # in parts
    need = _size("log_probs", p)[1]
    for i in range(7):  # logits, tokens, log_prob, entropy, stats, top_log_prob, top_token
        for bad in (None, P + 1):
            a = [P] * 7
            a[i] = bad
            assert lib.came8_log_probs_forward(ctypes.byref(p), *a, P, need, None) == L.CAME8_EINVAL
            if bad is None and i in (4, 5):
                continue
            assert lib.came8_log_probs_backward(ctypes.byref(p), *a, None) == L.CAME8_EINVAL  # ..., dlog_prob, dentropy, dlogits
    assert lib.came8_log_probs_backward(ctypes.byref(p), P, P, P, P, None, None, P, None) == L.CAME8_EINVAL
    for ws, size in ((None, need), (P + 8, need), (P, need - 1)):
        assert lib.came8_log_probs_forward(ctypes.byref(p), P, P, P, P, P, P, P, ws, size, None) == L.CAME8_ESPACE
    none = _desc(L.Came8LogProbs, PROBS, rows=0)
    assert lib.came8_log_probs_forward(ctypes.byref(none), *[None] * 8, 0, None) == L.CAME8_OK
    assert lib.came8_log_probs_backward(ctypes.byref(none), *[None] * 8) == L.CAME8_OK


def _calls():
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.long)
    q, s = torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    return {"embedding": (came_amd.embedding, [t, x]), "rms_norm": (came_amd.rms_norm, [x, x[0]]),
            "rms_norm_int8": (came_amd.rms_norm_int8, [x, x[0]]), "quantize_rows": (came_amd.quantize_rows, [x]),
            "int8_linear": (came_amd.int8_linear, [q, s, q, s]), "token_log_probs": (came_amd.token_log_probs, [x, t])}


@pytest.mark.parametrize("name", sorted(_calls()))
def test_cpu_tensors_and_others_raise(name):
    fn, args = _calls()[name]
    with pytest.raises(RuntimeError, match=f"{name}.*on the GPU"):
        fn(*args)
    for bad in (None, 3, [1.0]):
        with pytest.raises(RuntimeError, match="on the GPU"):
            fn(bad, *args[1:])


@pytest.mark.parametrize("name", sorted(_calls()))
def test_traces_and_tangents_are_refused(name):
    fn, args = _calls()[name]
    with pytest.raises(RuntimeError, match=f"{name}.*trace"):
        torch.jit.trace(lambda x: fn(x, *args[1:]), (args[0],), check_trace=False)
    k = next(i for i, a in enumerate(args) if a.is_floating_point())
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match=f"{name}.*({'on the GPU' if name == 'int8_linear' else 'tangent'})"):
        fn(*[forward_ad.make_dual(a, torch.ones_like(a)) if i == k else a for i, a in enumerate(args)])


def test_arguments_beside_the_tensors():
    t, w = torch.zeros(3, dtype=torch.long), torch.zeros(4, 8)
    for padding in (4, -5):
        with pytest.raises(ValueError, match="padding_idx"):
            came_amd.embedding(t, w, padding_idx=padding)
    q, s = torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    for dtype in (torch.int8, torch.float64, None):
        with pytest.raises(ValueError, match="dtype"):
            came_amd.int8_linear(q, s, q, s, dtype=dtype)
    with pytest.raises(TypeError):
        came_amd.rms_norm(w, w[0], eps="small")
    with pytest.raises(TypeError):
        came_amd.token_log_probs(w, t, top=1.5)


# ------------------------------------------------------------------------------------------------- the oracle
def test_oracle_gradients():
    gen = torch.Generator().manual_seed(0)
    d = dict(generator=gen, dtype=torch.float64)
    x, r, w, dy, dh = (torch.randn(*s, **d) for s in ((5, 7), (5, 7), (7,), (5, 7), (5, 7)))
    eps = float(torch.tensor(1e-3))
    a, b, c = (t.clone().requires_grad_() for t in (x, w, r))
    h = a + c
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * b
    want = torch.autograd.grad((y, h), (a, b), (dy, dh))
    for t in orc.UNIT:  # bounds of a type are the only thing that goes by it
        orc.rounded(torch.zeros(1), torch.zeros(1), t)
    (dx, _), (dw, _) = orc.rms_norm_gradients(h, w, 1e-3, dy.to(torch.float64).float().double().float(), dh.float())
    assert torch.allclose(dx, want[0], rtol=1e-5, atol=1e-5) and torch.allclose(dw, want[1], rtol=1e-5, atol=1e-5)
    z = torch.randn(6, 11, **d).requires_grad_()
    tokens = torch.randint(0, 11, (6,), generator=gen)
    tokens[2] = -100
    g, gh = torch.randn(6, **d), torch.randn(6, **d)
    logp = torch.log_softmax(z, -1)
    lp = torch.where(tokens >= 0, logp[torch.arange(6), tokens.clamp_min(0)], 0.0)
    entropy = -(logp.exp() * logp).sum(-1)
    (got, _), (H, _), kept = orc.log_probs(z, tokens)
    dz, _ = orc.log_probs_gradient(kept, g, gh, torch.float32)
    assert torch.allclose(got, lp) and torch.allclose(H, entropy)
    assert torch.allclose(dz, torch.autograd.grad((lp, entropy), z, (g, gh))[0])
    table = torch.randn(9, 4, **d).requires_grad_()
    t = torch.randint(0, 9, (20,), generator=gen)
    dy = torch.randn(20, 4, **d).float()
    want, = torch.autograd.grad(torch.nn.functional.embedding(t, table, padding_idx=3) * 2.0, table, dy.double())
    assert torch.allclose(orc.embedding_gradient(t, dy, 9, 2.0, 3)[0], want)


def test_oracle_codes():
    """Every code is the nearest to x * 127 / max, ties to even, found by comparing with all of them in whole numbers."""
    from fractions import Fraction
    gen = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(4, 30, generator=gen), (torch.randint(-127, 127, (3, 30), generator=gen) + 0.5)], 0)
    x[4:, 0] = 127.0
    q, s = orc.quantize_rows(x)
    for row, codes in zip(x.tolist(), q.tolist()):
        top = max(Fraction(abs(v)) for v in row)
        for v, c in zip(row, codes):
            e = Fraction(v) * 127 / top
            best = min(range(-127, 128), key=lambda k: (abs(e - k), k % 2))
            assert c == best, (v, c, best)
    assert torch.allclose(s, x.double().abs().amax(-1) / 127)
