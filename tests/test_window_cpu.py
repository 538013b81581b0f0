"""CPU tests of the windowed operators' argument checks. Nothing here launches a kernel."""
import ctypes

import pytest
import torch

import paged_attention as pa
from paged_attention import _native


def _decode_args():
    q = torch.randn(1, 2, 128, dtype=torch.float16)
    k = torch.randn(2, 16, 2, 128, dtype=torch.float16)
    return q, k, k, torch.zeros(1, 2, dtype=torch.int32), 16, 16


@pytest.mark.parametrize("kw,match", [
    (dict(window=0), "window must be at least 1"),
    (dict(window=-5), "window must be at least 1"),
    (dict(window=8, num_sinks=-1), "num_sinks must not be negative"),
    (dict(num_sinks=2), "num_sinks goes with a window"),
])
def test_window_arguments_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        pa.paged_attention(*_decode_args(), **kw)


def test_window_with_grad_is_inference_only():
    q, k, v, bt, s, bs = _decode_args()
    q.requires_grad_()
    with pytest.raises(RuntimeError, match="inference-only"):
        pa.paged_attention(q, k, v, bt, s, bs, window=4)


def test_sinks_without_a_window_are_refused_with_grad_too():
    q, k, v, bt, s, bs = _decode_args()
    q.requires_grad_()
    with pytest.raises(ValueError, match="num_sinks goes with a window"):
        pa.paged_attention(q, k, v, bt, s, bs, num_sinks=4)


def _params(**kw):
    p = _native.DecodeParams()
    p.batch, p.num_heads, p.num_kv_heads, p.head_dim = 2, 8, 2, 128
    p.block_size, p.num_blocks, p.max_blocks, p.seq_len = 16, 8, 4, 50
    p.scale, p.dtype = 0.088, _native.PA_F16
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,window,sinks,code", [
    ({}, 0, 0, _native.PA_ERR_ARG),
    ({}, -1, 0, _native.PA_ERR_ARG),
    ({}, 16, -1, _native.PA_ERR_ARG),
    ({"num_splits": 2}, 16, 0, _native.PA_ERR_UNSUPPORTED),
    ({"head_dim": 96}, 16, 0, _native.PA_ERR_UNSUPPORTED),
    ({"num_heads": 6, "num_kv_heads": 4}, 16, 0, _native.PA_ERR_ARG),
    ({"seq_len": 65}, 16, 0, _native.PA_ERR_ARG),
])
def test_window_c_abi_refusals(kw, window, sinks, code):
    lib = _native.lib()
    p = _params(**kw)
    a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert lib.pa_window_decode_workspace(ctypes.byref(p), window, sinks, ctypes.byref(a),
                                          ctypes.byref(b)) == code
    assert lib.pa_window_decode(ctypes.byref(p), window, sinks, None) == code


def test_window_c_abi_lengths_that_reach_int32s_end_are_refused():
    lib = _native.lib()
    p = _params(block_size=1024, max_blocks=2 ** 21, seq_len=2 ** 31 - 64)
    assert lib.pa_window_decode(ctypes.byref(p), 100, 4, None) == _native.PA_ERR_UNSUPPORTED
    p.seq_len = 2 ** 31 - 65                               # not refused for that
    assert lib.pa_window_decode(ctypes.byref(p), 100, 4, None) == _native.PA_ERR_ARG


def test_window_c_abi_null():
    lib = _native.lib()
    assert lib.pa_window_decode(None, 4, 0, None) == _native.PA_ERR_ARG
    assert lib.pa_window_decode(ctypes.byref(_params()), 4, 0, None) == _native.PA_ERR_ARG


def test_workspace_keeps_what_a_captured_graph_may_hold():
    import weakref
    ws = pa.DecodeWorkspace("cpu")
    ws.ensure(100, 10)
    held = [weakref.ref(ws.buffer), weakref.ref(ws.counters)]
    ws.ensure(1000, 100)
    ws.ensure(5000, 100)
    assert all(x() is not None for x in held)
    assert ws.buffer.numel() == 5000 and ws.counters.numel() == 100
    assert sum(x.numel() * x.element_size() for x in ws._earlier) <= 5000 + 400


def _prompt_args():
    q = torch.randn(3, 2, 128, dtype=torch.float16)
    k = torch.randn(2, 16, 2, 128, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    return q, k, k, torch.zeros(1, 2, dtype=torch.int32), i, i[:1], 16


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA tensors"),
    (dict(window=0), "window must be at least 1"),
    (dict(window=8, num_sinks=-1), "num_sinks must not be negative"),
    (dict(num_sinks=2), "num_sinks goes with a window"),
    (dict(num_splits=0), "num_splits must be at least 1"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
])
def test_prompt_arguments_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        pa.paged_prompt_attention(*_prompt_args(), **kw)


def test_prompt_with_grad_is_inference_only():
    args = _prompt_args()
    args[0].requires_grad_()
    with pytest.raises(RuntimeError, match="inference-only"):
        pa.paged_prompt_attention(*args)


def _prompt_params(**kw):
    p = _native.PromptParams()
    p.num_tokens, p.batch, p.num_heads, p.num_kv_heads, p.head_dim = 6, 2, 8, 2, 128
    p.block_size, p.num_blocks, p.max_blocks = 16, 8, 4
    p.scale, p.dtype = 0.088, _native.PA_F16
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,code", [
    ({}, _native.PA_ERR_ARG),                                     # null pointers
    ({"num_heads": 6, "num_kv_heads": 4}, _native.PA_ERR_ARG),
    ({"num_tokens": -1}, _native.PA_ERR_ARG),
    ({"batch": -1}, _native.PA_ERR_ARG),
    ({"dtype": 5}, _native.PA_ERR_ARG),
    ({"scale": 0.0}, _native.PA_ERR_ARG),
    ({"window": -1}, _native.PA_ERR_ARG),
    ({"num_sinks": 1}, _native.PA_ERR_ARG),
    ({"window": 4, "num_sinks": -1}, _native.PA_ERR_ARG),
    ({"num_splits": -1}, _native.PA_ERR_ARG),
    ({"head_dim": 96}, _native.PA_ERR_UNSUPPORTED),
    ({"max_blocks": 1 << 28}, _native.PA_ERR_UNSUPPORTED),
    ({"num_tokens": 1 << 28}, _native.PA_ERR_UNSUPPORTED),
])
def test_prompt_c_abi_refusals(kw, code):
    lib = _native.lib()
    assert lib.pa_prompt(ctypes.byref(_prompt_params(**kw)), None) == code
    assert lib.pa_prompt(None, None) == _native.PA_ERR_ARG


def test_prompt_c_abi_with_nothing_to_do():
    lib = _native.lib()
    for kw in ({"num_tokens": 0}, {"batch": 0}):
        assert lib.pa_prompt(ctypes.byref(_prompt_params(**kw)), None) == _native.PA_OK


def test_prompt_struct_layout_matches_header(tmp_path):
    import os
    import shutil
    import subprocess
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc not available")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cls, cname = _native.PromptParams, "pa_prompt_params"
    fields = [f[0] for f in cls._fields_]
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "pa_decode.h"',
           'int main(void) {', f'printf("size %zu\\n", sizeof({cname}));']
    src += [f'printf("{f} %zu\\n", offsetof({cname}, {f}));' for f in fields]
    src += ["return 0;", "}"]
    c = tmp_path / "probe.c"
    c.write_text("\n".join(src))
    exe = tmp_path / "probe"
    cuda_inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.run([gcc, "-I", os.path.join(root, "include"), "-I", cuda_inc, str(c), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    got = dict(line.split() for line in out.strip().splitlines())
    assert int(got["size"]) == ctypes.sizeof(cls)
    for f in fields:
        assert int(got[f]) == getattr(cls, f).offset, f
