"""Rows of a table, products by group and clipped steps together, as a program uses them: the example with layers of every element's own,
and a small head whose gradients and steps are held against the same formulas in 64 bits."""
import importlib.util
import math
import os

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("element_head", os.path.join(ROOT, "examples", "element_head.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _plain(leaves, descriptors, element):
    """The head in 64 bits; element: int64, -1 for none."""
    weight, bias, table, layer, layer_bias, readout, shift = leaves
    x = torch.nn.functional.layer_norm(descriptors, descriptors.shape[-1:], weight, bias, 1e-5)
    y = torch.zeros(len(element), dtype=torch.float64, device=element.device)
    for g in range(len(table)):
        at = (element == g).nonzero()[:, 0]
        h = torch.nn.functional.silu((x[at] + table[g]) @ layer[g].t() + layer_bias[g])
        y = y.index_put((at,), h @ readout[g, 0] + shift[g, 0])
    return y


def _doubles(tensors):
    return [t.detach().double().requires_grad_() for t in tensors]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_example_runs(example, dtype):
    first, last, norms, (head, descriptors, element, system) = example.run(steps=5, count=6, dtype=getattr(torch, dtype), quiet=True)
    assert all(math.isfinite(v) for v in (first, last, *norms)) and len(norms) == 5
    if dtype != "float32":
        return
    # its gradients, against the formulas': products of 64 terms and sums over up to 240 atoms, each off by less than (terms) 2^-24 of the sum of
    # the terms' sizes, which is taken as 64 times the largest gradient of the tensor; 512 covers both, and the layer norm's
    dy = torch.randn(len(system), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    mine = [p.grad for p in head.parameters()]
    assert all(g is not None for g in mine)
    got = torch.autograd.grad(head(descriptors, element), head.parameters(), dy)
    leaves = _doubles(head.parameters())
    want = torch.autograd.grad(_plain(leaves, descriptors.double(), element.index.long()), leaves, dy.double())
    for g, w in zip(got, want):
        assert ((g.double() - w).abs() <= 512 * 2.0 ** -24 * 64 * w.abs().max()).all()


class _Head:
    def __init__(self, d, hidden, elements, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s: torch.randn(*s, generator=g, device="cuda") * 0.3          # noqa: E731
        self.leaves = [1 + normal(d), normal(d), normal(elements, d), normal(elements, hidden, d), normal(elements, hidden), normal(elements, 1, hidden),
                       normal(elements, 1)]

    def __call__(self, descriptors, element):
        from symmetrix_amd import finetune as f
        weight, bias, table, layer, layer_bias, readout, shift = self.leaves
        x = f.layer_norm(descriptors, weight, bias) + f.embedding(table, element)
        return f.grouped_linear(torch.nn.functional.silu(f.grouped_linear(x, layer, layer_bias, element)), readout, shift, element)[:, 0]


def _batch(rows, d, elements, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    element = torch.randint(-1, elements, (rows,), generator=g, device="cuda", dtype=torch.int32)          # (some rows without one)
    return torch.randn(rows, d, generator=g, device="cuda"), element, torch.randn(rows, generator=g, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 1, 50, 700])
def test_steps_of_a_head(rows):
    """Three steps of forward, gradient and clipped AdamW, each from what the kernels' own step left."""
    from symmetrix_amd import finetune
    d, hidden, elements, max_norm, lr = 24, 40, 5, 0.25, 1e-2
    head = _Head(d, hidden, elements, rows)
    params = [p.requires_grad_() for p in head.leaves]
    opt = finetune.AdamW(params, lr=lr, weight_decay=0.0)
    moments = [(torch.zeros_like(p, dtype=torch.float64), torch.zeros_like(p, dtype=torch.float64)) for p in params]
    for step in range(1, 4):
        x, element, dy = _batch(rows, d, elements, step)
        groups = finetune.group_rows(element, elements)
        leaves, before = _doubles(params), [p.detach().double() for p in params]
        want = torch.autograd.grad(_plain(leaves, x.double(), element.long()), leaves, dy.double()) if rows else [torch.zeros_like(q) for q in leaves]
        for p in params:
            p.grad = None
        head(x, groups).backward(dy)
        for p, w in zip(params, want):
            # (as above: up to 700 rows, the terms of a sum up to 64 times its largest)
            assert ((p.grad.double() - w).abs() <= 1024 * 2.0 ** -24 * 64 * w.abs().max()).all()
        norm = opt.step(max_norm=max_norm)
        true = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
        assert abs(float(norm) - true) <= 2.0 ** -23 * true
        factor = min(1.0, max_norm / true) if true else 1.0
        for p, b, (m, v) in zip(params, before, moments):
            g = p.grad.double() * factor
            m.mul_(0.9).add_(g, alpha=0.1)
            v.mul_(0.999).addcmul_(g, g, value=0.001)
            u = lr * (m / (1 - 0.9 ** step)) / ((v / (1 - 0.999 ** step)).sqrt() + 1e-8)
            # the parameter's rounding; a number of the order of 1 of the update, whose moments take up to 6 roundings a step and whose
            # sum m may cancel to a tenth of its terms and less: an absolute part of the largest update that there can be, lr
            assert ((p.detach().double() - (b - u)).abs() <= 2.0 ** -24 * b.abs() + 64 * 2.0 ** -24 * lr + 1e-12).all()


@pytest.mark.gpu
def test_gradients_against_differences():
    """dL / dt along a direction, by five points of the head in 64 bits, against the kernels' gradient."""
    head = _Head(12, 20, 4, 3)
    x, element, dy = _batch(90, 12, 4, 4)
    params = [p.requires_grad_() for p in head.leaves]
    got = torch.autograd.grad(head(x, element), params, dy)
    base = [p.detach().double() for p in params]
    g = torch.Generator(device="cuda").manual_seed(9)
    for k, p in enumerate(base):
        along = torch.randn(p.shape, generator=g, device="cuda", dtype=torch.float64)
        loss = lambda t: float((_plain(base[:k] + [p + t * along] + base[k + 1:], x.double(), element.long()) * dy.double()).sum())          # noqa: E731,B023
        h = 1e-3
        slope = (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)
        # differences of fourth order: h^4 times a fifth derivative (of silu's arguments up to 4 along a direction of size 4, below 10^4 a row) over 30;
        # single precision: 1024 2^-24 of the terms
        assert abs(float((got[k].double() * along).sum()) - slope) <= 1024 * 2.0 ** -24 * float((got[k].double() * along).abs().sum()) + 1e-12 * 1e4 * 90


@pytest.mark.gpu
def test_a_captured_step_of_gradients():
    """Forward and backward in a graph, each replay against the eager result, with eager work between."""
    from symmetrix_amd import finetune
    d, elements, rows = 32, 6, 300
    head = _Head(d, 48, elements, 1)
    x, element, dy = _batch(rows, d, elements, 2)
    params = [p.requires_grad_() for p in head.leaves]

    def run():
        groups = finetune.group_rows(element, elements)
        return [*torch.autograd.grad(head(x, groups), params, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
        norm = finetune.clip_grads(got, 0.5)
    for k in range(4):
        new = _batch(rows, d, elements, 10 + k)
        for a, b in zip((x, element, dy), new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        mine, n = [t.clone() for t in got], norm.clone()
        want = run()
        true = finetune.clip_grads(want, 0.5)
        assert torch.equal(n, true) and all(torch.equal(a, b) for a, b in zip(mine, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_clipped_steps_with_masters(dtype):
    """Masters go by the clipped gradient in single precision, parameters are their roundings."""
    from symmetrix_amd import finetune
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(5)
    one = [torch.randn(n, generator=g, device="cuda").to(dtype) for n in (1000, 33, 4097)]
    two = [p.clone() for p in one]
    a, b = finetune.AdamW(one, lr=1e-2, masters=True), finetune.AdamW(two, lr=1e-2, masters=True)
    for k in range(3):
        grads = [torch.randn(p.shape, generator=g, device="cuda").to(dtype) for p in one]
        norm = math.sqrt(math.fsum(float(x.double().square().sum()) for x in grads))
        assert abs(float(a.step(grads, max_norm=2.0)) - norm) <= 2.0 ** -23 * norm
        factor = torch.tensor(2.0 / norm, dtype=torch.float32, device="cuda")
        b.step([x.float() * factor for x in grads])
        for p, q, m, n in zip(one, two, a.masters, b.masters):
            assert torch.equal(p, q) and torch.equal(m, n) and torch.equal(p, m.to(dtype))
