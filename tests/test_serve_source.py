"""What the serving kernels' source has to hold to, where no run on a GPU can show it: read here, on the CPU."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xlns-ggml-backend_b200", "csrc")


def _text(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _body(text, at):
    """from the first { behind `at` to its }"""
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[start:i]
    raise AssertionError("no end")


SERVE = _text("lnsb_serve.cu")
KERNELS = {m.group(1): (m.start(1), m) for m in re.finditer(
    r"__global__\s+void\s+(?:__launch_bounds__\([^)]*\)\s+)?(k_\w+)\(", SERVE)}


def test_kernels_are_found():
    assert sorted(KERNELS) == ["k_paged_append", "k_paged_append_vec", "k_paged_attn_rows", "k_paged_attn_tiles", "k_sample"]
    assert SERVE.count("__global__") == len(KERNELS)


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_every_kernel_waits_before_it_reads(name):
    """each is launched while the grid before it may still run: only behind its own wait, on every path, does it see
    what that grid and the ones before it wrote"""
    body = _body(SERVE, KERNELS[name][0])
    assert body.count("pdl_entry();") == 1
    lines = body[:body.index("pdl_entry();")].splitlines()
    assert lines[-1].strip() == ""                          # a statement of its own: behind no condition
    before = "\n".join(lines)
    assert before.count("{") - before.count("}") == 1       # in the kernel's outermost block
    for read in ("span_of(", "page_of(", "P.table", "P.q_start", "P.kv_len", "tma_page(", "__ldg(", "R.read("):
        for m in re.finditer(re.escape(read), before):
            # a lambda that is called later may stand before the wait
            inside = [l for l in re.finditer(r"auto\s+(\w+)\s*=\s*\[&\]", before)
                      if l.start() < m.start() < l.start() + len(_body(before, l.start())) + before.index("{", l.start()) - l.start()]
            assert inside, (name, read)
    assert "griddepcontrol" not in body
