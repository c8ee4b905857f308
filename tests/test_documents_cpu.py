"""The Python examples of the integration guide: they parse, and no module that an example imports is bound to something
else further down, so that its lines can be run in the order in which they stand."""
import ast
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def blocks():
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    return re.findall(r"```python\n(.*?)```", text, re.S)


@pytest.mark.parametrize("code", blocks(), ids=lambda c: c.strip().splitlines()[0][:40])
def test_examples_keep_the_modules_that_they_import(code):
    tree = ast.parse(code.replace("…", "..."))
    modules = {(a.asname or a.name).split(".")[0] for n in ast.walk(tree) if isinstance(n, (ast.Import, ast.ImportFrom)) for a in n.names}
    bound = {n.id for n in ast.walk(tree) if isinstance(n, ast.Name) and isinstance(n.ctx, ast.Store)}
    assert not modules & bound, modules & bound


def test_layers_of_the_example_exist():
    from bw1000_dsv4_kernels_b200 import ffn, moe, tp_linear
    modules = {"ffn": ffn, "moe": moe, "tp_linear": tp_linear}
    seen = 0
    for code in blocks():
        for n in ast.walk(ast.parse(code)):
            if isinstance(n, ast.Attribute) and isinstance(n.value, ast.Name) and n.value.id in modules:
                assert hasattr(modules[n.value.id], n.attr), f"{n.value.id}.{n.attr}"
                seen += 1
    assert seen >= 7
