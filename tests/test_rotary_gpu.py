"""GPU: rotary positions with several axes against the 64-bit formula, and their gradients.

Tolerance: an output is rounded once, by half a step of its type at most; before that it is ``x1 c - x2 s`` in fp32.
The angle's part below a turn is rounded to fp32 (half a turn at most: pi 2^-24 off), ``sincospif`` is exact to 2 units of
2^-24 of 1, the product and the FMA add 2^-24 each: below (pi + 2 + 2) 2^-24 < 5e-7 of ``|x1| + |x2|``.
"""

import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _tolerance(ref, x, R, dtype):
    turned = torch.zeros_like(ref)
    pair = x[..., :R].double().abs() + x[..., R: 2 * R].double().abs()
    turned[..., : 2 * R] = torch.cat([pair, pair], -1) * 5e-7
    least = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return ref.abs() * torch.finfo(dtype).eps / 2 * (1 + 1e-3) + turned * (1 + torch.finfo(dtype).eps) + least


def _inputs(B, H, H_kv, T, D, R, sections, dtype, far, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(B, h, T, D, generator=g).to(dtype) for h in (H, H_kv))
    positions = torch.randint(-far, far + 1, (len(sections), B, T), generator=g)
    inv_freq = 10000.0 ** (-torch.arange(R, dtype=torch.float64) / R)
    return q, k, positions, inv_freq


@pytest.mark.parametrize("B,H,H_kv,T,D,sections,dtype,far,pos_dtype", [
    (2, 4, 2, 37, 64, (32,), BF16, 5000, torch.int32),
    (3, 32, 8, 1, 128, (16, 24, 24), BF16, 1000000, torch.int32),       # one token per stream
    (1, 2, 2, 300, 64, (8, 12, 12), F16, 2**31 - 1, torch.int32),       # the farthest 32-bit positions, negative ones too
    (2, 3, 1, 65, 128, (64,), F32, 2**40, torch.int64),                 # farther still
    (1, 1, 1, 1, 16, (8,), F32, 10, torch.int64),
    (2, 5, 5, 33, 256, (64, 64), BF16, 4096, torch.int32),
    (2, 4, 4, 50, 128, (16, 16), BF16, 4096, torch.int32),              # half of the head is not rotated
    (2, 2, 2, 19, 64, (5, 2, 6), F16, 4096, torch.int32),               # an odd number of pairs: no vectors
    (1, 2, 2, 7, 32, (0, 16), F32, 100, torch.int32),                   # an axis without frequencies
    (1, 1, 1, 9, 32, (1,), BF16, 100, torch.int32),
    (1, 2, 1, 40, 64, (4,) * 8, F16, 1000, torch.int32),                # eight axes
    (70000, 1, 1, 1, 16, (8,), F16, 1000, torch.int32),                 # more sequences than a grid's second dimension
])
def test_rotary_matches_formula(B, H, H_kv, T, D, sections, dtype, far, pos_dtype):
    from kernels_b200.streaming_attention import rotary_embedding

    R = sum(sections)
    q, k, positions, inv_freq = _inputs(B, H, H_kv, T, D, R, sections, dtype, far)
    got = rotary_embedding(q.cuda(), k.cuda(), positions.to(pos_dtype).cuda(), inv_freq.cuda(), sections)
    if far > 2**31:
        # 2^40 radians in fp64 are off by 2^-13: the reference takes the part below a turn exactly
        from fractions import Fraction

        two_pi = Fraction("6.28318530717958647692528676655900576839433879875021164194988918461563281257")
        turns = [Fraction(float(f)) / two_pi for f in inv_freq]
        small = torch.empty(R, *positions.shape[1:], dtype=torch.float64)
        for d in range(R):
            for b in range(B):
                for t in range(T):
                    x = int(positions[0, b, t]) * turns[d]
                    small[d, b, t] = float((x - (x.numerator // x.denominator)) * two_pi)
        # (one axis per frequency with the reduced angle as its position and frequency 1)
        ref = [PO.rotary(x, small, torch.ones(R), (1,) * R) for x in (q, k)]
        slack = far * 2**-51  # the kernel's frequency in turns is a product in fp64 of two numbers of 53 bits
    else:
        ref = [PO.rotary(x, positions, inv_freq, sections) for x in (q, k)]
        # the reference's own angle in fp64, and the kernel's 53-bit frequency: p 2^-52 radians each
        slack = 2 * far * 2**-52
    for x, y, r in zip((q, k), got, ref):
        assert y.dtype == dtype and y.is_contiguous()
        pair = x.double().abs().max() * 2
        assert ((y.cpu().double() - r).abs() <= _tolerance(r, x, R, dtype) + slack * pair).all()
        assert torch.equal(y.cpu()[..., 2 * R:], x[..., 2 * R:])


def test_rotary_takes_any_layout_and_broadcast_positions():
    from kernels_b200.streaming_attention import rotary_embedding

    q, k, positions, inv_freq = _inputs(2, 4, 2, 21, 64, 32, (16, 16), F16, 500)
    qs = q.transpose(1, 2).contiguous().cuda().transpose(1, 2)               # [B, T, H, D] underneath
    ks = torch.zeros(2, 2, 21, 65, dtype=F16, device="cuda")[..., 1:]         # rows off the 16-byte boundaries
    ks.copy_(k)
    same = positions[:, :1].expand(2, 2, 21)
    want = rotary_embedding(q.cuda(), k.cuda(), same.contiguous().cuda(), inv_freq.cuda(), (16, 16))
    for pos in (positions[:, 0].cuda(), positions[:, :1].cuda().expand(2, 2, 21), positions[:, 0].t().contiguous().cuda().t()):
        for a, b in ((qs, ks), (q.cuda(), ks), (qs, k.cuda())):
            got = rotary_embedding(a, b, pos, inv_freq.cuda(), (16, 16))
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    alone = rotary_embedding(qs, None, positions[:, 0].cuda(), inv_freq.cuda(), (16, 16))
    assert alone[1] is None and torch.equal(alone[0], want[0])
    flipped = q.cuda().transpose(2, 3).contiguous().transpose(2, 3)           # D is not the inner axis
    assert torch.equal(rotary_embedding(flipped, None, positions[:, 0].cuda(), inv_freq.cuda(), (16, 16))[0], want[0])


def test_rotary_empty_calls():
    from kernels_b200.streaming_attention import rotary_embedding

    f = torch.ones(8, dtype=torch.float64, device="cuda")
    for B, H, T in ((0, 2, 3), (2, 0, 3), (2, 2, 0)):
        x = torch.zeros(B, H, T, 16, device="cuda")
        y, z = rotary_embedding(x, x, torch.zeros(1, B, T, dtype=torch.int32, device="cuda"), f)
        assert y.shape == x.shape and z.shape == x.shape
    q, k = torch.randn(2, 2, 3, 16, device="cuda"), torch.randn(2, 0, 3, 16, device="cuda")
    y, z = rotary_embedding(q, k, torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda"), f)
    assert torch.equal(y, q) and z.shape == k.shape
    y, z = rotary_embedding(k, q, torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda"), f)
    assert torch.equal(z, q) and y.shape == k.shape


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rotary_gradient_is_the_opposite_turn(dtype):
    from kernels_b200.streaming_attention import rotary_embedding

    sections, R = (4, 6, 6), 16
    q, k, positions, inv_freq = _inputs(2, 4, 2, 33, 64, R, sections, dtype, 2000, seed=1)
    gq, gk = _inputs(2, 4, 2, 33, 64, R, sections, dtype, 10, seed=2)[:2]
    qc, kc = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    y = rotary_embedding(qc, kc, positions.cuda(), inv_freq.cuda(), sections)
    dq, dk = torch.autograd.grad(y, (qc, kc), (gq.cuda(), gk.cuda().transpose(1, 2).contiguous().transpose(1, 2)))
    for g, d in ((gq, dq), (gk, dk)):
        ref = PO.rotary(g, -positions, inv_freq, sections)
        assert ((d.cpu().double() - ref).abs() <= _tolerance(ref, g, R, dtype) + 4000 * 2**-52 * 20).all()


def test_rotary_gradient_against_differences():
    """fp32, central differences of a weighted sum: the operator is linear, so they are exact up to rounding.  The sum has
    768 terms of about 1 in fp64 over fp32 outputs, each off by 5e-7 (|x1| + |x2|) < 5e-6 at a step of 1: far below 1e-4."""
    from kernels_b200.streaming_attention import rotary_embedding

    sections = (3, 5)
    q, _, positions, inv_freq = _inputs(1, 2, 1, 12, 32, 8, sections, F32, 50, seed=3)
    g = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).double()
    qc = q.cuda().requires_grad_()
    f = lambda x: (rotary_embedding(x, None, positions.cuda(), inv_freq.cuda(), sections)[0].double().cpu() * g).sum()  # noqa: E731
    (dq,) = torch.autograd.grad(f(qc), qc)
    for i in ((0, 0, 0, 0), (0, 1, 7, 9), (0, 1, 11, 15), (0, 0, 3, 31), (0, 1, 5, 2)):
        e = torch.zeros_like(q)
        e[i] = 1.0
        with torch.no_grad():
            slope = (f((q + e).cuda()) - f((q - e).cuda())) / 2
        assert abs(float(slope) - float(dq[i])) < 1e-4


def test_rotary_second_gradients_and_unused_outputs():
    from kernels_b200.streaming_attention import rotary_embedding

    sections = (8,)
    q, k, positions, inv_freq = (x.cuda() for x in _inputs(1, 2, 2, 5, 16, 8, sections, F32, 9))
    q.requires_grad_(), k.requires_grad_()
    y, _ = rotary_embedding(q, k, positions, inv_freq)
    (dq,) = torch.autograd.grad(y.square().sum() / 2, q, create_graph=True)
    assert torch.allclose(dq, q, atol=1e-5)  # a rotation's transpose undoes it
    (again,) = torch.autograd.grad(dq.square().sum() / 2, q)
    assert torch.allclose(again, q, atol=1e-5)
    # the keys alone, the queries alone, gradients that come expanded
    for grads in ((False, True), (True, False)):
        x, y = q.detach().requires_grad_(grads[0]), k.detach().requires_grad_(grads[1])
        out = rotary_embedding(x, y, positions, inv_freq)
        leaf, got = (x, out[0]) if grads[0] else (y, out[1])
        (d,) = torch.autograd.grad((out[0] + out[1]).sum(), leaf)
        ref = PO.rotary(torch.ones_like(leaf.cpu().detach()), -positions.cpu(), inv_freq.cpu(), sections)
        assert torch.allclose(d.cpu().double(), ref, atol=1e-5) and got.requires_grad
    (d,) = torch.autograd.grad(rotary_embedding(q, None, positions, inv_freq)[0].sum(), q)
    assert d.shape == q.shape


def test_rotary_under_transforms():
    """Forward-mode tangents and functorch gradients turn with the tensors; a compiled caller gets the eager result."""
    import torch.autograd.forward_ad as fw
    from kernels_b200.streaming_attention import rotary_embedding

    sections = (4, 12)
    q, k, positions, inv_freq = (x.cuda() for x in _inputs(2, 2, 1, 9, 64, 16, sections, F32, 50))
    t = torch.randn_like(q)
    want = rotary_embedding(q, k, positions, inv_freq, sections)
    with fw.dual_level():
        y, z = rotary_embedding(fw.make_dual(q, t), k, positions, inv_freq, sections)
        y, tangent = fw.unpack_dual(y)
        z, none = fw.unpack_dual(z)
        assert torch.equal(y, want[0]) and torch.equal(z, want[1]) and (none is None or (none == 0).all())
        assert torch.equal(tangent, rotary_embedding(t, None, positions, inv_freq, sections)[0])
    g = torch.func.grad(lambda x: (rotary_embedding(x, None, positions, inv_freq, sections)[0] * t).sum())(q)
    x = q.clone().requires_grad_()
    (ref,) = torch.autograd.grad(rotary_embedding(x, None, positions, inv_freq, sections)[0], x, t)
    assert torch.equal(g, ref)
    compiled = torch.compile(lambda x, y: rotary_embedding(x * 1, y, positions, inv_freq, sections))
    assert all(torch.equal(a, b) for a, b in zip(compiled(q, k), want))


def _second_inputs(sections, seed):
    return [x.cuda() for x in _inputs(2, 4, 2, 17, 64, sum(sections), sections, F32, 500, seed=seed)]


@pytest.mark.parametrize("keys", [True, False])
@pytest.mark.parametrize("grad", [False, True])
def test_rotary_is_recorded_by_whatever_traces(keys, grad):
    """A traced function computes on the tensors that it is called with, with gradients and without."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from kernels_b200.streaming_attention import rotary_embedding

    sections = (8, 24)

    def turn(q, k, positions, inv_freq):
        y, z = rotary_embedding(q, k if keys else None, positions, inv_freq, sections)
        return (y, z) if keys else (y,)

    first, second = _second_inputs(sections, 1), _second_inputs(sections, 2)
    if grad:
        first[0].requires_grad_(), first[1].requires_grad_(), second[0].requires_grad_(), second[1].requires_grad_()
    want = turn(*second)
    traced = {
        "jit.trace": lambda: torch.jit.trace(turn, tuple(first), check_trace=False), "make_fx": lambda: make_fx(turn)(*first),
        "make_fx, fake": lambda: make_fx(turn, tracing_mode="fake")(*first), "compile": lambda: torch.compile(turn, fullgraph=True),
    }
    for what, trace in traced.items():
        got = trace()(*second)
        got = got if isinstance(got, (tuple, list)) else (got,)
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), what
        if grad and what in ("jit.trace", "compile"):
            leaves = second[: len(want)]
            g = [torch.randn(x.shape, generator=torch.Generator().manual_seed(5)).cuda() for x in want]
            a, b = torch.autograd.grad(got, leaves, g), torch.autograd.grad(turn(*second), leaves, g)
            assert all(torch.equal(x, y) for x, y in zip(a, b)), what


def test_rotary_under_modes_and_subclasses():
    from torch.utils._python_dispatch import TorchDispatchMode
    from kernels_b200.streaming_attention import rotary_embedding

    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    class Sub(torch.Tensor):
        pass

    q, k, positions, inv_freq = _second_inputs((32,), 3)
    want = rotary_embedding(q, k, positions, inv_freq)
    with Mode():
        got = rotary_embedding(q, k, positions, inv_freq)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and any("rotary" in s for s in seen)
    got = rotary_embedding(q.as_subclass(Sub), k, positions, inv_freq)
    assert all(torch.equal(a.as_subclass(torch.Tensor), b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError):  # no rule for batches of calls
        torch.func.vmap(lambda x: rotary_embedding(x, None, positions, inv_freq)[0])(q[None])
    x = q.clone().requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
        (d,) = torch.autograd.grad(rotary_embedding(x, k, positions, inv_freq)[0], x, q)
    assert torch.equal(d, torch.autograd.grad(rotary_embedding(x, k, positions, inv_freq)[0], x, q)[0])
    (d,) = torch.autograd.grad(torch.ops.kernels_b200.rotary_embedding(x, None, positions, inv_freq, [32], False)[0], x, q, create_graph=True)
    assert torch.equal(d, torch.autograd.grad(rotary_embedding(x, None, positions, inv_freq)[0], x, q)[0]) and d.requires_grad is False


def test_rotary_gradients_of_transforms_are_recorded_too():
    from torch.fx.experimental.proxy_tensor import make_fx
    from kernels_b200.streaming_attention import rotary_embedding

    q, k, positions, inv_freq = _second_inputs((32,), 3)
    t, other = torch.randn_like(q), torch.randn_like(q)
    loss = lambda x, y: (rotary_embedding(x, None, y, inv_freq)[0] * t).sum()  # noqa: E731
    leaf = q.clone().requires_grad_()
    (want,) = torch.autograd.grad(loss(leaf, positions), leaf)
    grad = torch.func.grad(loss)
    assert torch.equal(grad(q, positions), want)
    assert torch.equal(make_fx(grad)(other, positions.flip(-1))(q, positions), want)
    assert torch.equal(torch.compile(grad)(q, positions), want)
    tangent = lambda x, d: torch.func.jvp(lambda z: rotary_embedding(z, None, positions, inv_freq)[0], (x,), (d,))[1]  # noqa: E731
    turned = rotary_embedding(t, None, positions, inv_freq)[0]
    assert torch.equal(tangent(q, t), turned) and torch.equal(torch.compile(tangent)(q, t), turned)


@pytest.mark.parametrize("keys", [True, False])
def test_rotary_operator_is_what_it_says(keys):
    """Schema, fake form, gradient and compiled form agree with the operator; a compiled caller takes other lengths."""
    from kernels_b200.streaming_attention import rotary_embedding

    q, k, positions, inv_freq = _second_inputs((8, 24), 4)
    q.requires_grad_(), k.requires_grad_()
    torch.library.opcheck(torch.ops.kernels_b200.rotary_embedding.default, (q, k if keys else None, positions, inv_freq, [8, 32], False))
    compiled = torch.compile(lambda q, k, p: rotary_embedding(q, k if keys else None, p, inv_freq, (8, 24)), fullgraph=True, dynamic=True)
    for T in (17, 5, 1):
        args = (q[:, :, :T], k[:, :, :T], positions[:, :, :T])
        got, want = compiled(*args), rotary_embedding(args[0], args[1] if keys else None, args[2], inv_freq, (8, 24))
        assert torch.equal(got[0], want[0]) and (torch.equal(got[1], want[1]) if keys else got[1] is None)


def test_rotary_of_lazily_negated_tensors():
    """The imaginary part of a conjugate carries its sign as a mark on the tensor: inputs, frequencies, gradients and tangents alike."""
    from kernels_b200.streaming_attention import rotary_embedding

    q, k, positions, inv_freq = (x.cuda() for x in _inputs(2, 4, 2, 17, 64, 32, (32,), F32, 500))

    def marked(x):
        y = torch.complex(torch.zeros_like(x), -x).conj().imag
        assert y.is_neg() and torch.equal(y, x)
        return y

    want = rotary_embedding(q, k, positions, inv_freq)
    for change in (dict(q=marked(q)), dict(k=marked(k)), dict(inv_freq=marked(inv_freq))):
        got = rotary_embedding(**(dict(q=q, k=k, positions=positions, inv_freq=inv_freq) | change))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), tuple(change)
    x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
    out = rotary_embedding(x, y, positions, inv_freq)
    plain = torch.autograd.grad(out, (x, y), (q, k), retain_graph=True)
    got = torch.autograd.grad(out, (x, y), (marked(q), marked(k)))
    assert all(torch.equal(a, b) for a, b in zip(got, plain))


def test_rotary_in_a_graph_and_on_another_stream():
    from kernels_b200.streaming_attention import rotary_embedding

    q, k, positions, inv_freq = (x.cuda() for x in _inputs(2, 4, 2, 17, 64, 32, (32,), BF16, 500))
    want = rotary_embedding(q, k, positions, inv_freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotary_embedding(q, k, positions, inv_freq)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x, pos = torch.empty_like(q), torch.zeros_like(positions)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = rotary_embedding(x, k, pos, inv_freq)
    x.copy_(q), pos.copy_(positions)
    graph.replay()
    assert torch.equal(y, want[0])


def test_rotary_backward_in_a_graph():
    """Forward and gradient captured together (no eager graph of the same leaf is alive: torch ends the process then, whatever the operator)."""
    from kernels_b200.streaming_attention import rotary_embedding

    q, _, positions, inv_freq = (x.cuda() for x in _inputs(2, 4, 2, 17, 64, 32, (32,), BF16, 500))
    g = torch.randn_like(q)
    leaf = torch.zeros_like(q).requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = rotary_embedding(leaf, None, positions, inv_freq)
        (d,) = torch.autograd.grad(y, leaf, g)
    with torch.no_grad():
        leaf.copy_(q)
    for scale in (1.0, -2.0):
        g.copy_(torch.randn_like(g) * scale)
        graph.replay()
        assert torch.equal(y, rotary_embedding(q, None, positions, inv_freq)[0])
        assert torch.equal(d, rotary_embedding(g, None, -positions, inv_freq)[0])


def test_rotary_refusals():
    from kernels_b200.streaming_attention import rotary_embedding

    q, k, positions, inv_freq = (x.cuda() for x in _inputs(2, 4, 2, 17, 64, 32, (32,), BF16, 500))
    bad = [
        dict(positions=positions.float()), dict(positions=positions[:, :1]), dict(positions=positions[0, 0]), dict(inv_freq=inv_freq.float()),
        dict(sections=(16, 16)), dict(sections=(31,)), dict(sections=(33, -1), positions=positions.expand(2, 2, 17)), dict(k=k.half()),
        dict(k=k[:1]), dict(inv_freq=torch.ones(33, dtype=torch.float64, device="cuda")), dict(positions=positions.cpu()),
        dict(positions=positions.expand(9, 2, 17), sections=(32,) + (0,) * 8), dict(inv_freq=inv_freq.clone().requires_grad_()),
    ]
    for change in bad:
        args = dict(q=q, k=k, positions=positions, inv_freq=inv_freq) | change
        with pytest.raises(AssertionError):
            rotary_embedding(**args)
    with pytest.raises(RuntimeError, match="unsupported"):
        rotary_embedding(q.double(), None, positions, inv_freq)
    with pytest.raises(RuntimeError, match="unsupported"):
        rotary_embedding(q[..., :48], None, positions, inv_freq[:24])
