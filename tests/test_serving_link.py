"""Refusals of the operators over a paged cache and of the choice of tokens that need no GPU, and the restatements that the GPU tests compare with."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from ocannl_b200 import backend as bk
from tests import serving_reference as R
from tests.test_operators_link import context

BF = "bfloat16"


def test_specs_have_the_layout_of_the_header(built_lib, tmp_path):
    """The ctypes mirrors against sizes and offsets that a C compiler gives."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    specs = {"b200_cache": bk.CacheSpec, "b200_cache_append": bk.CacheAppendSpec, "b200_cache_attention": bk.CacheAttentionSpec, "b200_sample": bk.SampleSpec}
    lines = []
    for c, py in specs.items():
        lines.append('printf("%s %%zu", sizeof(%s));' % (c, c))
        lines += ['printf(" %%zu", offsetof(%s, %s));' % (c, f) for f, _ in py._fields_]
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
    for entry, spec in (("b200_cache_append_link", bk.CacheAppendSpec()), ("b200_cache_attention_link", bk.CacheAttentionSpec()), ("b200_sample_link", bk.SampleSpec())):
        assert getattr(bk.lib(), entry)(None, ctypes.byref(spec), ctypes.byref(out)) == -1
        assert "null" in bk.lib().b200_last_error().decode()


CACHE = ("k_cache", "v_cache")


@pytest.mark.parametrize("call,words", [
    (lambda c: c.cache_append("none", "v", *CACHE, "pages", "lens"), "no node 'none'"),
    (lambda c: c.cache_append("logits", "v", *CACHE, "pages", "lens"), "[tokens, heads, d]"),
    (lambda c: c.cache_append("k", "q", *CACHE, "pages", "lens"), "dims"),
    (lambda c: c.cache_append("k", "v", "k", "v_cache", "pages", "lens"), "[pages, kv_heads, page, 16]"),
    (lambda c: c.cache_append("q", "q", *CACHE, "pages", "lens"), "heads, the cache"),
    (lambda c: c.cache_append("k", "v", *CACHE, "lens", "lens"), "[batch, max_pages]"),
    (lambda c: c.cache_append("k", "v", *CACHE, "pages", "pages"), "dims"),
    (lambda c: c.cache_append("k", "v", *CACHE, "pages", "lens", starts="lens"), "dims"),
    (lambda c: c.cache_append("k", "v", *CACHE, "pages", "lens", k_scale="scale"), "go together"),
    (lambda c: c.cache_append("k", "v", *CACHE, "pages", "lens", k_scale="scale", v_scale="scale"), "precision"),
    (lambda c: c.cache_append("k", "v", "codes", "codes", "pages", "lens"), "precision"),
    (lambda c: c.cache_append("k", "v", "codes", "codes", "pages", "lens", k_scale="u", v_scale="u"), "dims"),
    (lambda c: c.cache_append("k", "v", *CACHE, "pages", "lens", q="q"), "go together"),
    (lambda c: c.cache_append("k", "v", *CACHE, "pages", "lens", q="q", q_out="k"), "dims"),
    (lambda c: c.cache_append("k", "v", *CACHE, "pages", "lens", layout="other"), "layout"),
    (lambda c: c.cache_append("k", "v", *CACHE, "pages", "lens", positions="lens"), "dims"),
    (lambda c: c.cache_attention("logits", *CACHE, "q", "pages", "lens"), "[tokens, heads, d]"),
    (lambda c: c.cache_attention("q", *CACHE, "k", "pages", "lens"), "dims"),
    (lambda c: c.cache_attention("q", "k_cache", "codes", "q2", "pages", "lens"), "precision"),
    (lambda c: c.cache_attention("q", *CACHE, "q2", "pages", "lens", lse="u"), "dims"),
    (lambda c: c.cache_attention("q", *CACHE, "q2", "pages", "lens", slopes="u"), "dims"),
    (lambda c: c.cache_attention("q", *CACHE, "q2", "none", "lens"), "no node 'none'"),
    (lambda c: c.sample("ids", "u", "ids"), "precision"),
    (lambda c: c.sample("logits", "ids", "ids"), "precision"),
    (lambda c: c.sample("logits", "u", "lens"), "dims"),
    (lambda c: c.sample("logits", "u", "ids", top_k="u"), "precision"),
    (lambda c: c.sample("logits", "u", "ids", temperature="scale"), "dims"),
    (lambda c: c.sample("logits", "u", "ids", logprob="ids"), "precision"),
])
def test_nodes_are_checked(call, words):
    c = context(q=(BF, (6, 4, 16)), q2=(BF, (6, 4, 16)), k=(BF, (6, 2, 16)), v=(BF, (6, 2, 16)), k_cache=(BF, (9, 2, 8, 16)), v_cache=(BF, (9, 2, 8, 16)),
                codes=("byte", (9, 2, 8, 16)), scale=("single", (9, 2)), pages=("int32", (3, 4)), lens=("int32", (3,)), starts=("int32", (4,)),
                logits=(BF, (5, 100)), u=("single", (5,)), ids=("int32", (5,)))
    with pytest.raises(bk.UserError) as e:
        call(c)
    assert words in str(e.value)


def test_codes_of_the_restatement():
    fine = [c for c in range(256) if c & 127 != 127]
    assert all(int(R.encode(R.E4M3[c])) == c for c in fine if R.E4M3[c] != 0)
    assert R.E4M3[0x7e] == 448.0 and R.E4M3[1] == 2.0 ** -9 and R.E4M3[8] == 2.0 ** -6
    # halfway: to the even one; beyond the last: to it
    assert R.decode(R.encode([17.0, 19.0, 500.0, 2.0 ** -10, 3 * 2.0 ** -10])).tolist() == [16.0, 20.0, 448.0, 0.0, 2.0 ** -8]
    assert [R.exponent(a) for a in (0.0, 448.0, 448.0001, 1.0, 3.6)] == [-40, 0, 1, -8, -6]


def test_choice_of_the_restatement():
    x = np.log([0.1, 0.4, 0.2, 0.2, 0.1])
    assert R.sample(x, 0.0) == (0, pytest.approx(np.log(0.1))) and R.sample(x, 0.999)[0] == 4
    assert R.sample(x, 0.5, top_k=1) == (1, 0.0) and R.sample(x, 0.7, top_k=2)[0] == 2
    # ties: the lower index is kept
    assert [R.sample(x, u, top_k=2)[0] for u in (0.0, 0.6, 0.99)] == [1, 1, 2]
    assert [R.sample(x, 0.99, top_p=p)[0] for p in (0.0, 0.39, 0.41, 0.61, 0.81)] == [1, 1, 2, 3, 3]
    assert [R.sample(x, 0.99, min_p=p)[0] for p in (0.0, 0.4, 0.6, 2.0)] == [4, 3, 1, 1]
    assert R.sample([np.nan, -np.inf], 0.5) == (-1, -np.inf) and R.sample([1.0, np.inf, np.inf, np.nan], 0.6)[0] == 2
    assert R.sample([3.0, 5.0, 5.0], 0.9, temperature=0.0) == (1, 0.0)
