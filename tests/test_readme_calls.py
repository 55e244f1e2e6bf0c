"""The README's calls of the fine-tuning operators are calls that can be made."""
import ast
import inspect
import os
import re

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _block():
    with open(os.path.join(ROOT, "README.md")) as f:
        blocks = re.findall(r"```python\n(.*?)```", f.read(), re.S)
    return next(b for b in blocks if "import finetune" in b)


def test_arguments_are_in_order():
    """Every call binds to its function, and an argument that has a parameter's name stands in that parameter's place."""
    from symmetrix_amd import finetune
    seen = 0
    for node in ast.walk(ast.parse(_block())):
        if isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute) and getattr(node.func.value, "id", "") == "finetune":
            bound = inspect.signature(getattr(finetune, node.func.attr)).bind(*node.args, **{k.arg: k.value for k in node.keywords})
            names = list(inspect.signature(getattr(finetune, node.func.attr)).parameters)
            for name, value in bound.arguments.items():
                assert not isinstance(value, ast.Name) or value.id not in names or value.id == name
            seen += 1
    assert seen >= 3


@pytest.mark.gpu
def test_the_block_runs():
    g = torch.Generator(device="cuda").manual_seed(0)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")          # noqa: E731
    names = dict(descriptors=normal(50, 64), weight=torch.ones(64, device="cuda", requires_grad=True), bias=torch.zeros(64, device="cuda", requires_grad=True),
                 W=normal(32, 64), A=normal(3, 4, 64).requires_grad_(), B=normal(3, 32, 4).requires_grad_(), scale=torch.ones(3, device="cuda"),
                 index=(torch.arange(50, device="cuda") % 4 - 1).to(torch.int32))
    exec(_block(), names)
    names["y"].square().sum().backward()
    before = names["A"].detach().clone()
    names["opt"].step()
    assert names["y"].shape == (50, 32) and not torch.equal(names["A"], before)
