"""Refusals of the sink adapter and its library entry points, on the CPU."""

import ctypes

import pytest
import torch

import gemma4_fa4_amd as g4
from gemma4_fa4_amd import _lib


def args():
    bf = dict(dtype=torch.bfloat16)
    c = torch.tensor([0, 8], dtype=torch.int32)
    return dict(q=torch.zeros(8, 32, 256, **bf), k=torch.zeros(8, 16, 256, **bf),
                v=torch.zeros(8, 16, 256, **bf), cu_seqlens_q=c, cu_seqlens_k=c,
                max_seqlen_q=8, max_seqlen_k=8, num_sinks=4)


@pytest.mark.parametrize("change,error,match", [
    (dict(num_sinks=True), TypeError, "integer"),
    (dict(num_sinks=2.0), TypeError, "integer"),
    (dict(num_sinks=-1), g4.UnsupportedMI355XPath, "num_sinks"),
    (dict(num_sinks=33), g4.UnsupportedMI355XPath, "num_sinks"),
    (dict(q=torch.zeros(8, 32, 256)), ValueError, "BF16"),
    (dict(spec=g4.GLOBAL_ATTENTION), ValueError, "spec"),
    (dict(max_seqlen_q=9, max_seqlen_k=9), ValueError, "maxima"),
    (dict(max_seqlen_q=9), g4.UnsupportedMI355XPath, "max Sq <= max Sk"),
    ({}, g4.UnsupportedMI355XPath, "GPU tensors"),
])
def test_adapter_arguments(change, error, match):
    a = args() | change
    with pytest.raises(error, match=match):
        g4.fa4_local_sinks_varlen_forward(**a)


def problem(**change):
    p = dict(num_seqs=1, seqlen_q=2048, seqlen_k=2048, num_q_heads=32, num_kv_heads=16,
             head_dim=256, window=1024, total_q=2048, total_k=2048)
    return _lib.G4Problem(**(p | change))


@pytest.mark.parametrize("change,sinks,rc", [
    (dict(head_dim=512), 4, _lib.G4_ERR_UNSUPPORTED), (dict(window=0), 4, _lib.G4_ERR_UNSUPPORTED),
    ({}, 0, _lib.G4_ERR_UNSUPPORTED), ({}, 33, _lib.G4_ERR_UNSUPPORTED),
    (dict(num_seqs=0), 4, _lib.G4_ERR_INVALID),
    (dict(vision_ids=64), 4, _lib.G4_ERR_UNSUPPORTED),
    (dict(document_ids=64), 4, _lib.G4_ERR_UNSUPPORTED),
])
def test_the_library_refuses(change, sinks, rc):
    lib = _lib.load()
    p = problem(**change)
    assert lib.g4_sinks_workspace_bytes(ctypes.byref(p), sinks, 1) == 0 and lib.g4_last_error()
    lay = _lib.G4Layout(0, 8192, 256)
    x = 4096
    assert lib.g4_attn_sinks_fwd(ctypes.byref(p), sinks, x, lay, x, lay, x, lay, x, lay, x, x, 0,
                                 None) == rc
    assert lib.g4_attn_sinks_bwd(ctypes.byref(p), sinks, x, lay, x, lay, x, lay, x, lay, x, lay, x,
                                 None, x, lay, x, lay, x, lay, x, 0, None) == rc


def test_workspaces():
    lib = _lib.load()
    p = problem()
    ref = ctypes.byref(p)
    assert lib.g4_sinks_workspace_bytes(ref, 4, 0) == 0 and lib.g4_last_error() == b""
    base = lib.g4_workspace_bytes(ref, 1)
    need = lib.g4_sinks_workspace_bytes(ref, 4, 1)
    # the chunks' dK and dV: at least one 32-key block of each per KV head
    assert need - base >= 16 * 2 * 32 * 256 * 4
    lay, x = _lib.G4Layout(0, 8192, 256), 4096
    call = lambda ws, n: lib.g4_attn_sinks_bwd(  # noqa: E731
        ref, 4, x, lay, x, lay, x, lay, x, lay, x, lay, x, None, x, lay, x, lay, x, lay, ws, n, None)
    assert call(x, need - 1) == _lib.G4_ERR_WORKSPACE
    assert call(None, need) == _lib.G4_ERR_WORKSPACE
    assert call(x + 16, need) == _lib.G4_ERR_WORKSPACE
    step = problem(seqlen_q=1, total_q=1)
    need = lib.g4_sinks_workspace_bytes(ctypes.byref(step), 4, 0)
    assert need > 0
    assert lib.g4_attn_sinks_fwd(ctypes.byref(step), 4, x, lay, x, lay, x, lay, x, lay, x, x,
                                 need - 1, None) == _lib.G4_ERR_WORKSPACE
