"""RowGroups after writes: their tensors are addresses of rows, and have to be those that the index was sorted into."""
import pytest

torch = pytest.importorskip("torch")


def _groups(device="cpu"):
    from symmetrix_amd import finetune
    index = torch.tensor([2, 0, -1, 2], dtype=torch.int32, device=device)
    return finetune.RowGroups(index, 3, torch.tensor([1, 0, 3, 2], dtype=torch.int32, device=device), torch.tensor([0, 1, 1, 3, 4], dtype=torch.int32, device=device))


@pytest.mark.parametrize("which", ["index", "order", "offsets"])
def test_written_to(which):
    groups = _groups()
    assert groups.of(3) is groups
    with pytest.raises(ValueError):
        groups.of(4)
    getattr(groups, which).add_(1)
    with pytest.raises(ValueError, match="written to"):
        groups.of(3)


def test_made_by_hand():
    from symmetrix_amd import finetune
    g = _groups()
    for order, offsets in ((g.order[:3], g.offsets), (g.order, g.offsets[:4]), (g.order.long(), g.offsets), (g.order, g.offsets.float()),
                           (torch.zeros(8, dtype=torch.int32)[::2], g.offsets)):
        with pytest.raises(ValueError):
            finetune.RowGroups(g.index, 3, order, offsets)
    with torch.inference_mode():
        uncounted = g.index.clone()
    for tensors in ((uncounted, g.order, g.offsets), (g.index, uncounted, g.offsets)):
        with pytest.raises(ValueError, match="inference"):
            finetune.RowGroups(tensors[0], 3, *tensors[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("inside", [True, False])
@pytest.mark.parametrize("rows", [50, 100, 700])
def test_indices_of_inference_mode(rows, inside):
    """Calls by RowGroups go by what the index held when its rows were sorted, all of them; order and offsets count their versions."""
    from symmetrix_amd import finetune
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, w, b, dy = (torch.randn(*s, generator=g, device="cuda") for s in ((rows, 40), (5, 24, 40), (5, 24), (rows, 24)))
    first, second = (torch.randint(-1, 5, (rows,), generator=g, device="cuda", dtype=torch.int32) for _ in range(2))
    with torch.inference_mode():
        index = first.clone()
    assert index.is_inference()

    def calls(i):
        return [finetune.grouped_linear_forward(x, w, b, i), *finetune.grouped_linear_backward(dy, x, w, i), finetune.embedding_forward(w[:, 0], i, 2.0),
                finetune.embedding_backward(dy, i, 5)]

    with torch.inference_mode(inside):
        groups = finetune.group_rows(index, 5)
        want = calls(first)
        for a, c in zip(calls(groups), want):
            assert torch.equal(a, c)
    with torch.inference_mode():
        index.copy_(second)
        for a, c in zip(calls(groups), want):
            assert torch.equal(a, c)
    leaf = w.clone().requires_grad_()
    finetune.grouped_linear(x, leaf, b, groups).backward(dy)
    assert torch.equal(leaf.grad, want[2])
    groups.order.mul_(1)
    with pytest.raises(ValueError, match="written to"):
        finetune.grouped_linear_forward(x, w, b, groups)


@pytest.mark.gpu
def test_ordinary_indices_in_inference_mode():
    from symmetrix_amd import finetune
    index = torch.tensor([2, 0, -1, 2], dtype=torch.int32, device="cuda")
    with torch.inference_mode():
        groups = finetune.group_rows(index, 3)
        assert groups.index is index and groups.order.tolist() == [1, 0, 3, 2] and groups.offsets.tolist() == [0, 1, 1, 3, 4]
        table = torch.ones(3, 8, device="cuda")
        assert finetune.embedding_forward(table, groups).sum() == 24
        index.add_(0)
        with pytest.raises(ValueError, match="written to"):
            finetune.embedding_forward(table, groups)
