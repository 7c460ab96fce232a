"""Refusals of the operators' link entry points that need no GPU: arguments are checked before anything is launched."""
import ctypes

import pytest

from ocannl_b200 import backend as bk
from ocannl_b200.low_level import Tnode


def test_specs_have_the_layout_of_the_header(built_lib, tmp_path):
    """The ctypes mirrors against sizes and offsets that a C compiler gives."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    specs = {"b200_layer_norm": bk.LayerNormSpec, "b200_rotary": bk.RotarySpec, "b200_attention": bk.AttentionSpec, "b200_operand": bk.Operand}
    lines = []
    for c, py in specs.items():
        lines.append('printf("%s %%zu", sizeof(%s));' % (c, c))
        for f, _ in py._fields_:
            lines.append('printf(" %%zu", offsetof(%s, %s));' % (c, f))
        lines.append('printf("\\n");')
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s/include/b200.h"\nint main(void){%s return 0;}\n' % (root, "\n".join(lines)))
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", str(src), "-o", exe], check=True)
    for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines():
        name, *numbers = line.split()
        py = specs[name]
        assert [int(n) for n in numbers] == [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_], name


def test_null_arguments(built_lib):
    out = ctypes.c_void_p()
    for entry, spec in (("b200_layer_norm_link", bk.LayerNormSpec()), ("b200_layer_norm_grad_link", bk.LayerNormSpec()), ("b200_rotary_link", bk.RotarySpec()),
                        ("b200_attention_link", bk.AttentionSpec()), ("b200_attention_grad_link", bk.AttentionSpec())):
        assert getattr(bk.lib(), entry)(None, ctypes.byref(spec), ctypes.byref(out)) == -1
        assert "null" in bk.lib().b200_last_error().decode()
    assert bk.lib().b200_operator_run(None) == -1
    assert bk.lib().b200_operator_free(None) == 0


class _NoDevice:
    h = None


def context(**nodes):
    """A context whose nodes are only described: what the Python side refuses needs no device."""
    arrays = {n: (1, 0, Tnode(i + 1, n, prec, dims)) for i, (n, (prec, dims)) in enumerate(nodes.items())}
    return bk.Context(_NoDevice(), arrays)


BF = "bfloat16"


@pytest.mark.parametrize("call,words", [
    (lambda c: c.layer_norm("none", "y"), "no node 'none'"),
    (lambda c: c.layer_norm("x", "short"), "dims"),
    (lambda c: c.layer_norm("x", "single"), "precision"),
    (lambda c: c.layer_norm("x", "y", gamma="gamma", beta="gamma_bf"), "one precision"),
    (lambda c: c.layer_norm("x", "y", gamma="stat"), "dims"),
    (lambda c: c.layer_norm("ids", "y"), "precision"),
    (lambda c: c.layer_norm_grad("x", "y", "dx", "stat", "gamma"), "dims"),
    (lambda c: c.rotary([("x", "y")], [1.0]), "[batch, seq, heads, d]"),
    (lambda c: c.rotary([], [1.0]), "one or two"),
    (lambda c: c.rotary([("q", "q2")] * 3, [1.0]), "one or two"),
    (lambda c: c.rotary([("q", "q2")], [1.0], layout="other"), "layout"),
    (lambda c: c.rotary([("q", "k")], [1.0]), "dims"),
    (lambda c: c.rotary([("q", "q2")], [1.0], positions="lens"), "dims"),
    (lambda c: c.attention("x", "k", "v", "q2"), "[batch, queries, heads, d]"),
    (lambda c: c.attention("q", "k", "v", "q2", mask="other"), "unknown mask"),
    (lambda c: c.attention("q", "k", "q", "q2"), "dims"),
    (lambda c: c.attention("q", "k", "v", "k"), "dims"),
    (lambda c: c.attention("q", "k", "v", "q2", lengths="stat"), "precision"),
    (lambda c: c.attention("q", "k", "v", "q2", documents="lens"), "dims"),
    (lambda c: c.attention("q", "k", "v", "q2", slopes="gamma"), "dims"),
])
def test_nodes_are_checked(call, words):
    c = context(x=(BF, (5, 8)), y=(BF, (5, 8)), dx=(BF, (5, 8)), short=(BF, (5, 7)), single=("single", (5, 8)), gamma=("single", (8,)), gamma_bf=(BF, (8,)),
                stat=("single", (5,)), ids=("int32", (5, 8)), q=(BF, (2, 3, 4, 16)), q2=(BF, (2, 3, 4, 16)), k=(BF, (2, 9, 2, 16)), v=(BF, (2, 9, 2, 16)),
                lens=("int32", (2,)))
    with pytest.raises(bk.UserError) as e:
        call(c)
    assert words in str(e.value)


def test_rotary_frequencies():
    f, m = bk.rotary_frequencies(64)
    assert m == 1.0 and f[0] == 1.0 and abs(f[31] - 10000.0 ** (-62 / 64)) < 1e-18
    g, _ = bk.rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert g[0] == 1.0 and abs(g[31] / f[31] * 8.0 - 1.0) < 1e-12
    y, m = bk.rotary_frequencies(64, scaling="yarn", factor=8.0)
    assert y[0] == f[0] and abs(y[31] / f[31] * 8.0 - 1.0) < 1e-12 and m > 1.0 and all(a > b for a, b in zip(y, y[1:]))
    assert bk.rotary_frequencies(0)[0].size == 0
    for bad in (dict(dims=63), dict(dims=64, scaling="unknown"), dict(dims=64, theta=0.0), dict(dims=64, factor=-1.0)):
        with pytest.raises(bk.UserError):
            bk.rotary_frequencies(**bad)
