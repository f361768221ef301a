"""What the serving calls refuse, and the arguments' layout: no GPU needed, the
checks come before any CUDA call."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, TOO_LARGE = -1, -4


@pytest.fixture(scope="module")
def lib():
    import build
    build.build_all(["base"])
    from lnsb200 import _lib
    return _lib.load("base")


def _kv():
    return dict(k_cache=4096, v_cache=8192, page_stride=16 * 2 * 64, row_stride=128, head_stride=64, page_table=64, q_start=64,
                kv_len=64, table_ld=4, n_pages=8, n_tokens=3, max_kv=64, n_seqs=2, type=1, page_size=16, n_head_kv=2,
                head_dim=64)


def _append(lib, **kw):
    from lnsb200 import _lib
    a = _lib.PagedAppendArgs(**{**_kv(), **dict(k=64, v=64, q=64, q_out=64, cos_sin=64, k_ld=128, v_ld=128, q_ld=256,
                                                q_out_ld=256, in_type=0, n_head=4, n_dims=64, neox=0), **kw})
    return lib.lnsb_paged_append(ctypes.byref(a), None)


def _attn(lib, **kw):
    from lnsb200 import _lib
    a = _lib.PagedAttnArgs(**{**_kv(), **dict(q=64, dst=64, work=64, work_bytes=1 << 40, q_ld=256, dst_ld=256, max_q=3,
                                              window=0, n_head=4, scale=0.125), **kw})
    return lib.lnsb_paged_attn(ctypes.byref(a), None)


def _sample(lib, **kw):
    from lnsb200 import _lib
    a = _lib.SampleArgs(**{**dict(logits=64, u=64, token=64, ld=100, n_rows=2, n_vocab=100, type=0), **kw})
    return lib.lnsb_sample(ctypes.byref(a), None)


KV_BAD = [dict(type=0), dict(type=8), dict(page_size=12), dict(page_size=4), dict(page_size=2048), dict(page_size=0),
          dict(head_dim=80), dict(head_dim=0), dict(n_head_kv=0), dict(n_seqs=-1), dict(n_tokens=-1), dict(n_pages=-1),
          dict(max_kv=65), dict(max_kv=-1), dict(row_stride=132), dict(head_stride=60), dict(page_stride=2052),
          dict(k_cache=4104), dict(v_cache=8194), dict(k_cache=None), dict(page_table=None), dict(q_start=None),
          dict(kv_len=None)]


@pytest.mark.parametrize("bad", KV_BAD, ids=str)
def test_paged_plan_refused(lib, bad):
    assert _append(lib, **bad) == INVALID
    assert _attn(lib, **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(cos_sin=None), dict(n_dims=63),
                                 dict(n_dims=66), dict(n_dims=-2), dict(in_type=2), dict(k_ld=127), dict(v_ld=127),
                                 dict(q_ld=255), dict(q_out_ld=255), dict(n_head=0), dict(n_head=-1)], ids=str)
def test_append_refused(lib, bad):
    assert _append(lib, **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(q=None), dict(dst=None), dict(work=None), dict(work_bytes=100), dict(n_head=3),
                                 dict(n_head=0), dict(q_ld=255), dict(q_ld=260), dict(dst_ld=252), dict(q=72), dict(dst=72),
                                 dict(work=72), dict(window=-1), dict(max_q=-1)], ids=str)
def test_attn_refused(lib, bad):
    assert _attn(lib, **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(logits=None), dict(u=None), dict(token=None), dict(n_vocab=0), dict(ld=99),
                                 dict(n_rows=-1), dict(type=2), dict(type=8)], ids=str)
def test_sample_refused(lib, bad):
    assert _sample(lib, **bad) == INVALID


def test_sizes_refused(lib):
    assert _append(lib, n_pages=1 << 32) == TOO_LARGE
    assert _attn(lib, table_ld=1 << 30, max_kv=1 << 31) == TOO_LARGE
    assert _attn(lib, n_seqs=65537) == TOO_LARGE
    assert _sample(lib, n_vocab=(1 << 20) + 1, ld=1 << 21) == TOO_LARGE


def test_nothing_to_do(lib):
    assert _append(lib, n_tokens=0) == 0 and _append(lib, n_seqs=0) == 0
    assert _attn(lib, n_tokens=0) == 0 and _attn(lib, n_seqs=0) == 0
    assert _sample(lib, n_rows=0) == 0
    assert lib.lnsb_paged_append(None, None) == INVALID
    assert lib.lnsb_paged_attn(None, None) == INVALID
    assert lib.lnsb_sample(None, None) == INVALID


def test_argument_layout(tmp_path):
    """the ctypes structures are the header's"""
    from lnsb200 import _lib
    src = tmp_path / "layout.c"
    names = {"lnsb_paged_append_args": _lib.PagedAppendArgs, "lnsb_paged_attn_args": _lib.PagedAttnArgs,
             "lnsb_sample_args": _lib.SampleArgs}
    kv = {n for n, _ in _lib._PAGED_KV}
    lines = ["#include <stdio.h>", '#include "lnsb200.h"', "int main(void) {"]
    for c, py in names.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (c, c))
        for f, _ in py._fields_:
            if f != "_pad":
                lines.append('printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (c, f, c, ("kv." + f) if f in kv and "paged" in c else f))
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = dict(l.split() for l in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    for c, py in names.items():
        assert int(got[c]) == ctypes.sizeof(py)
        for f, _ in py._fields_:
            if f != "_pad":
                assert int(got["%s.%s" % (c, f)]) == getattr(py, f).offset, (c, f)


def test_python_refusals():
    """shapes and types that the binding turns away"""
    import lnsb200
    ks = lnsb200.KernelSet(16, "base")
    kc, i32 = torch.zeros(4, 16, 2, 64, dtype=torch.float16), torch.int32
    table, q_start, kv_len = torch.zeros(1, 4, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32)
    k = torch.zeros(3, 2, 64)
    good = dict(k=k, v=k, k_cache=kc, v_cache=kc, page_table=table, q_start=q_start, kv_len=kv_len, max_kv=10)
    for bad in (dict(v=k.half()), dict(k=k[:, :1]), dict(k=k.double(), v=k.double()), dict(v_cache=kc.bfloat16()),
                dict(v_cache=kc[:2]), dict(page_table=table.long()), dict(kv_len=q_start), dict(q_start=kv_len),
                dict(cos_sin=torch.zeros(9, 32, 2)), dict(cos_sin=torch.zeros(10, 32, 2).half()),
                dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(3, 4, 64), q_out=torch.zeros(3, 4, 64)),
                dict(k=k.transpose(1, 2), v=k.transpose(1, 2))):
        with pytest.raises(ValueError):
            ks.paged_append(**{**good, **bad})
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    good = dict(q=q, k_cache=kc, v_cache=kc, page_table=table, q_start=q_start, kv_len=kv_len, max_q=3, max_kv=10, dst=q,
                work=torch.zeros(8))
    for bad in (dict(q=q.float()), dict(dst=q.bfloat16()), dict(dst=q[:2]), dict(q=q[..., :32], dst=q[..., :32])):
        with pytest.raises(ValueError):
            ks.paged_attn(**{**good, **bad})
    x, u = torch.zeros(2, 50), torch.zeros(2)
    for bad in (dict(logits=x.T), dict(logits=x.double()), dict(u=u.double()), dict(u=torch.zeros(3)),
                dict(token=torch.zeros(2, dtype=torch.int64)), dict(top_k=u), dict(temperature=torch.zeros(1))):
        with pytest.raises(ValueError):
            ks.sample(**{**dict(logits=x, u=u, token=torch.zeros(2, dtype=i32)), **bad})
