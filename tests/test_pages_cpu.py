"""CPU tests of the page operators' boundary: argument checks that need no GPU, the
struct layout, and the row-by-row model that the GPU tests compare with."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import paged_attention as pa
from page_model import NO_PAGES, PageModel
from paged_attention import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cpu_caches_refused():
    k = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA tensors"):
        pa.PagePool(k, k)
    with pytest.raises(ValueError, match="at least one layer"):
        pa.PagePool([], [])
    with pytest.raises(ValueError, match=r"\[num_blocks, block_size, Hkv, D\]"):
        pa.PagePool(k[0], k[0])


def _pool(**kw):
    p = _native.PagePoolParams()
    buf = ctypes.create_string_buffer(4096)
    p.refs = p.free_words = p.scratch = p.status = ctypes.addressof(buf)
    p.num_blocks, p.block_size, p.num_kv_heads, p.head_dim = 8, 16, 2, 64
    p.scratch_ints = 10 ** 6
    for k, v in kw.items():
        setattr(p, k, v)
    return p, buf


@pytest.mark.parametrize("kw,code", [
    ({"num_blocks": 0}, _native.PA_ERR_ARG),
    ({"block_size": 0}, _native.PA_ERR_ARG),
    ({"head_dim": 0}, _native.PA_ERR_ARG),
    ({"num_layers": -1}, _native.PA_ERR_ARG),
    ({"num_layers": 1, "caches": None}, _native.PA_ERR_ARG),
    ({"refs": None}, _native.PA_ERR_ARG),
    ({"free_words": None}, _native.PA_ERR_ARG),
    ({"scratch": None}, _native.PA_ERR_ARG),
    ({"k_stride_slot": 4}, _native.PA_ERR_ARG),
    ({"head_dim": 20}, _native.PA_ERR_UNSUPPORTED),
    ({"num_blocks": 1 << 30}, _native.PA_ERR_UNSUPPORTED),
    ({"scratch_ints": 63}, _native.PA_ERR_WORKSPACE),
])
def test_pool_struct_checked(kw, code):
    lib = _native.lib()
    p, buf = _pool(**kw)
    at = ctypes.addressof(buf)
    assert lib.pa_pages_resize(ctypes.byref(p), at, 4, 2, 4, at, at, 0, 0, None) == code
    assert lib.pa_pages_fork(ctypes.byref(p), at, 4, 2, 4, at, at, at, 1, None) == code
    assert lib.pa_pages_compact(ctypes.byref(p), at, 4, 2, 4, at, None) == code


def test_calls_checked():
    lib = _native.lib()
    p, buf = _pool()
    at, ref = ctypes.addressof(buf), ctypes.byref(p)
    bad = _native.PA_ERR_ARG
    assert lib.pa_pages_resize(None, at, 4, 2, 4, at, at, 0, 0, None) == bad
    assert lib.pa_pages_resize(ref, None, 4, 2, 4, at, at, 0, 0, None) == bad
    assert lib.pa_pages_resize(ref, at, 4, -1, 4, at, at, 0, 0, None) == bad
    assert lib.pa_pages_resize(ref, at, 4, 2, 4, None, at, 0, 0, None) == bad
    assert lib.pa_pages_resize(ref, at, 4, 2, 4, at, None, 0, 0, None) == bad
    assert lib.pa_pages_resize(ref, at, 4, 2, 4, at, at, -1, 0, None) == bad
    assert lib.pa_pages_resize(ref, at, 4, 2, 4, at, at, 0, 3, None) == bad
    assert lib.pa_pages_fork(ref, at, 4, 2, 4, at, None, at, 1, None) == bad
    assert lib.pa_pages_fork(ref, at, 4, 2, 4, at, at, at, -1, None) == bad
    assert lib.pa_pages_compact(ref, at, 4, 2, 4, None, None) == bad
    assert lib.pa_pages_scratch(ref, 2, 2, None) == bad
    assert lib.pa_pages_adopt(ref, at, 4, 2, 4, None, None) == bad
    assert lib.pa_pages_adopt(ref, None, 4, 2, 4, at, None) == bad
    assert lib.pa_pages_adopt(ref, at, 4, 2, -1, at, None) == bad
    # nothing to do: no launch, so this works without a GPU
    assert lib.pa_pages_resize(ref, at, 4, 0, 4, at, at, 0, 0, None) == _native.PA_OK
    assert lib.pa_pages_fork(ref, at, 4, 2, 4, at, at, at, 0, None) == _native.PA_OK


def test_struct_layout_matches_header(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc not available")
    cls, cname = _native.PagePoolParams, "pa_page_pool"
    fields = [f[0] for f in cls._fields_]
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "pa_decode.h"',
           'int main(void) {', f'printf("size %zu\\n", sizeof({cname}));']
    src += [f'printf("{f} %zu\\n", offsetof({cname}, {f}));' for f in fields]
    src += ["return 0;", "}"]
    c = tmp_path / "probe.c"
    c.write_text("\n".join(src))
    exe = tmp_path / "probe"
    cuda_inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.run([gcc, "-I", os.path.join(ROOT, "include"), "-I", cuda_inc, str(c), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    got = dict(line.split() for line in out.strip().splitlines())
    assert int(got["size"]) == ctypes.sizeof(cls)
    for f in fields:
        assert int(got[f]) == getattr(cls, f).offset, f


def test_model_frees_what_the_window_hides():
    """Pages of 4 tokens, window 6, 3 sinks: a row of 20 growing to 21 keeps the sinks'
    page and those from token 15 on; the free pages are taken from the lowest."""
    k = torch.zeros(8, 4, 1, 8)
    m = PageModel([k], [k], torch.full((2, 8), -1), torch.zeros(2, dtype=torch.int32))
    m.resize([20, 0])
    assert m.table[0][:5] == [0, 1, 2, 3, 4]
    m.resize([21, 0], 6, 3)
    assert m.table[0][:6] == [0, -1, -1, 3, 4, 1] and m.refs == [1, 1, 0, 1, 1, 0, 0, 0]
    m.resize([-1, 17])
    assert m.status == NO_PAGES and m.lens == [21, 0]


def test_int64_lengths_and_rows_are_not_wrapped():
    from paged_attention.page_pool import int32_vector
    x = int32_vector("who", torch.tensor([0, 5, -1, -2 ** 40, 2 ** 31 - 1, 2 ** 32 + 7]))
    assert x.dtype == torch.int32 and x.tolist() == [0, 5, -1, -1, 2 ** 31 - 1, 2 ** 31 - 1]
    y = torch.arange(6, dtype=torch.int32)
    assert int32_vector("who", y) is y and int32_vector("who", y[::2]).is_contiguous()
    for bad in (torch.zeros(2), torch.zeros(2, dtype=torch.int16)):
        with pytest.raises(ValueError, match="who: lengths and rows"):
            int32_vector("who", bad)
