"""GPU tests of the trainable grouped products: the forward product of any row length, autograd,
and the SwiGLU experts, against formulas in 64 bits and against differences."""
import pytest
import torch

from light_moe_b200 import ops
from light_moe_b200.grouped import GroupedExperts, GroupedLinear, grouped_linear

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _inputs(counts, n, k, dt, seed=0, tail=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b = [0]
    for c in counts:
        b.append(b[-1] + c)
    x = torch.randn(b[-1] + tail, k, generator=gen, device="cuda").to(dt)
    w = (torch.randn(len(counts), n, k, generator=gen, device="cuda") * 0.1).to(dt)
    return x, w, b, torch.tensor(b, device="cuda")


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("counts,n,k", [([3, 0, 40], 33, 1), ([130, 61], 64, 66), ([257, 5], 300, 200), ([1], 8, 264),
                                        ([70, 300, 0, 9], 517, 1409), ([40, 600], 1000, 72)])
def test_product_of_any_row_length(dt, counts, n, k):
    """L products summed in fp32 (L * 2^-23 of the absolute sum), one rounding to the type."""
    x, w, b, off = _inputs(counts, n, k, DT[dt], tail=3)
    x[b[-1]:] = float("nan")
    y = ops.grouped_gemm(x, w, off, len(counts))
    assert y.dtype == DT[dt] and (y[b[-1]:] == 0).all()
    half = torch.finfo(y.dtype).eps / 2
    for e in range(len(counts)):
        r = slice(b[e], b[e + 1])
        want, mass = x[r].double() @ w[e].double().T, x[r].double().abs() @ w[e].double().abs().T
        tol = (k + 1) * 2.0 ** -23 * mass * (1 + half) + half * want.abs() + torch.finfo(y.dtype).tiny
        assert ((y[r].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("n,k", [(96, 128), (33, 50)])
def test_gradients_against_differences(n, k):
    """The product is linear in each operand: <g, y(w + d) - y(w)> = <dw, d> for any step d, up to
    the fp32 sums' error (2^-23 per addition of what is added)."""
    x, w, b, off = _inputs([40, 0, 17, 70], n, k, torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(5)
    g, dx, dw = (torch.randn(*s, generator=gen, device="cuda") for s in ((b[-1], n), x.shape, w.shape))
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    grouped_linear(xl, wl, off).backward(g)
    y = grouped_linear(x, w, off).double()
    mass = grouped_linear(x.abs() + dx.abs(), w.abs() + dw.abs(), off).double()
    depth = max(n, k, 70)
    for step, grad, moved in ((dw, wl.grad, grouped_linear(x, w + dw, off)), (dx, xl.grad, grouped_linear(x + dx, w, off))):
        got = (grad.double() * step.double()).sum()
        want = (g.double() * (moved.double() - y)).sum()
        assert (got - want).abs() <= 4 * (depth + 2) * 2.0 ** -23 * (g.double().abs() * mass).sum()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_autograd_calls(dt):
    x, w, b, off = _inputs([30, 0, 33], 64, 128, DT[dt])
    x.requires_grad_()
    y = grouped_linear(x, w, off)
    y.sum().backward()                       # a broadcast gradient
    ones = torch.ones_like(y)
    assert torch.equal(x.grad, ops.grouped_gemm_dgrad(ones, w, off, 3)) and w.grad is None
    m = GroupedLinear(3, 128, 64, device="cuda", dtype=DT[dt])
    m(x.detach(), off).backward(ones)
    assert torch.equal(m.weight.grad, ops.grouped_gemm_wgrad(ones, x.detach(), off, 3))
    assert (m.weight.grad[1] == 0).all()
    shared = w[:1].clone().requires_grad_()  # one matrix for every expert: its gradients add up
    grouped_linear(x.detach(), shared.expand(3, -1, -1), off).backward(ones)
    want = ops.grouped_gemm_wgrad(ones, x.detach(), off, 3).sum(0, keepdim=True)
    assert torch.equal(shared.grad, want)
    z = grouped_linear(x, w, off)
    (g1,) = torch.autograd.grad(z, x, ones, create_graph=True)
    with pytest.raises(RuntimeError):        # differentiable once
        g1.sum().backward()


def test_refusals():
    x, w, b, off = _inputs([30, 33], 64, 128, torch.bfloat16)
    for call in (lambda: grouped_linear(x, w.float(), off), lambda: grouped_linear(x[0], w, off),
                 lambda: grouped_linear(x, w[:, :, :64], off), lambda: grouped_linear(x, w, off[:2]),
                 lambda: grouped_linear(x.double(), w.double(), off)):
        with pytest.raises(ValueError):
            call()


def _experts_reference(x, ids, wts, w1, w3, w2):
    y = torch.zeros_like(x)
    for j in range(ids.shape[1]):
        for e in range(w1.shape[0]):
            m = ids[:, j] == e
            xe = x[m]
            h = torch.nn.functional.silu(xe @ w1[e].T) * (xe @ w3[e].T)
            y = y.index_add(0, m.nonzero()[:, 0], (h @ w2[e].T) * wts[m, j][:, None])
    return y


@pytest.mark.parametrize("T,d,f,E,k", [(50, 64, 96, 4, 2), (1, 40, 33, 3, 3), (200, 128, 256, 8, 2)])
def test_experts_against_autograd_in_64_bits(T, d, f, E, k):
    """fp32 in every step.  `mass` is the same formula on absolute values: a bound on the sums of
    absolute terms up to what silu does to signs.  Each of the three products in a row is off by
    (depth + 1) * 2^-23 of its absolute sum and the elementwise steps by a few units; |silu'| <= 1.1
    while silu' >= 1/2 on the absolute side (a factor 2.2, rounded up to 4 with silu itself), and
    |silu''| <= 1/2 turns an error of the gate's sum, at most `reach` times the unit, into one of
    silu'."""
    gen = torch.Generator(device="cuda").manual_seed(T)
    m = GroupedExperts(E, d, f, device="cuda", dtype=torch.float32)
    x = torch.randn(T, d, generator=gen, device="cuda", requires_grad=True)
    ids = torch.rand(T, E, generator=gen, device="cuda").topk(k).indices
    if E > 3:
        ids[ids == 1] = 0                    # an expert without tokens, tokens with an expert twice
    wts = torch.rand(T, k, generator=gen, device="cuda", requires_grad=True)
    y = m(x, ids, wts)
    g = torch.randn(T, d, generator=gen, device="cuda")
    leaves = (x, wts, m.gate_proj.weight, m.up_proj.weight, m.down_proj.weight)
    got = torch.autograd.grad(y, leaves, g)
    ref = [t.detach().double().requires_grad_() for t in leaves]
    yr = _experts_reference(ref[0], ids, ref[1], *ref[2:])
    want = torch.autograd.grad(yr, ref, g.double())
    absr = [t.detach().double().abs().requires_grad_() for t in leaves]
    ya = _experts_reference(absr[0], ids, absr[1], *absr[2:])
    mass = torch.autograd.grad(ya, absr, g.double().abs())
    unit = 2.0 ** -23 * (3 * (max(d, f, T * k) + 1) + 32)
    reach = (absr[0] @ absr[2].flatten(0, 1).T).max().item()
    for a, b, c in zip((y,) + got, (yr,) + want, (ya,) + mass):
        assert ((a.double() - b).abs() <= 4 * (1 + reach) * unit * c.abs() + 1e-37).all()


def test_training_step_in_a_graph():
    """Forward and backward captured once and replayed on new data equal the eager step."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    T, d, f, E, k = 96, 128, 128, 4, 2
    m = GroupedExperts(E, d, f, device="cuda", dtype=torch.bfloat16)
    params = list(m.parameters())
    x = torch.randn(T, d, generator=gen, device="cuda").to(torch.bfloat16)
    ids = torch.rand(T, E, generator=gen, device="cuda").topk(k).indices
    wts = torch.rand(T, k, generator=gen, device="cuda")

    def step():
        y = m(x, ids, wts)
        return (y.detach(),) + torch.autograd.grad(y, params, torch.ones_like(y))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(x.flip(0) * 0.5)
    ids.copy_((ids + 1) % E)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_experts_without_tokens_and_with_odd_indices():
    m = GroupedExperts(3, 32, 64, device="cuda", dtype=torch.float32)
    x = torch.zeros(0, 32, device="cuda", requires_grad=True)
    ids, w = torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, 2, device="cuda")
    y = m(x, ids, w)
    y.sum().backward()
    assert y.shape == (0, 32) and x.grad.shape == (0, 32)
    assert all((p.grad == 0).all() for p in m.parameters())
    # the same expert twice counts twice; indices that name no expert add nothing
    x = torch.randn(5, 32, device="cuda")
    one = m(x, torch.full((5, 1), 2, device="cuda"), torch.ones(5, 1, device="cuda"))
    two = m(x, torch.full((5, 2), 2, device="cuda"), torch.full((5, 2), 0.5, device="cuda"))
    none = m(x, torch.tensor([[-1, 2, 3]], device="cuda").expand(5, 3), torch.ones(5, 3, device="cuda"))
    assert torch.equal(one, two) and torch.equal(one, none)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_sizes_beyond_32_bits_are_refused(dt):
    """A size is never cut to its lower 32 bits (2^32 + 5 would count as 5).  The operands are views of
    one value: nothing of that size is allocated."""
    one = torch.ones(1, device="cuda", dtype=DT[dt])
    off = torch.tensor([0, 1], device="cuda")
    big = 2 ** 32 + 5
    for x, w in ((one.view(1, 1), one.expand(1, big, 1)), (one.expand(1, big), one.expand(1, 1, big)),
                 (one.expand(big, 1), one.view(1, 1, 1))):
        with pytest.raises(RuntimeError, match="32 bits"):
            ops.grouped_gemm(x, w, off, 1)


@pytest.mark.parametrize("dt,k", [("bf16", 128), ("fp16", 128), ("fp32", 64), ("bf16", 130), ("fp32", 33)])
def test_operands_that_start_anywhere(dt, k):
    """Contiguous views one value behind an aligned address, forward and through autograd."""
    gen = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(5 * k + 1, generator=gen, device="cuda").to(DT[dt])[1:].view(5, k)
    w = torch.randn(2 * 24 * k + 1, generator=gen, device="cuda").to(DT[dt])[1:].view(2, 24, k)
    off = torch.tensor([0, 2, 5], device="cuda")
    want = ops.grouped_gemm(x.clone(), w.clone(), off, 2)
    assert torch.equal(ops.grouped_gemm(x, w, off, 2), want)
    xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = grouped_linear(xl, wl, off)
    y.sum().backward()
    assert torch.equal(y, want)
    assert torch.equal(xl.grad, ops.grouped_gemm_dgrad(torch.ones_like(y), w.clone(), off, 2))
    assert torch.equal(wl.grad, ops.grouped_gemm_wgrad(torch.ones_like(y), x.clone(), off, 2))
