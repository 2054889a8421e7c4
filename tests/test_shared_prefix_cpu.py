"""mgi_paged_decode_shared without a GPU: its refusals (every one returns before
any HIP call) and its workspace sizes."""
from __future__ import annotations

import ctypes

import pytest
import torch

from minivllm import _native
from minivllm import hip_paged_decode as hpd
from minivllm.kv_block_pool import KVBlockPool

P = ctypes.c_void_p(4096)  # never read: the calls are refused on the host


def _st(*s):
    return (ctypes.c_int64 * len(s))(*s)


CALL = dict(out=P, os=_st(512, 64, 1), q=P, qs=_st(512, 64, 1), kp=P, vp=P, kps=_st(8192, 2048, 128, 64, 1),
            vps=_st(8192, 2048, 128, 64, 1), dt=1, bt=P, bts=_st(8, 1), bti=1, cl=P, cls=1, cli=1, B=2, Hq=8, Hk=2, D=64,
            S=16, N=4, M=8, L=1, layer=0, shared=4, scale=0.125, ws=None, bytes=0, stream=None)


@pytest.mark.parametrize("change,code,msg", [
    (dict(out=None), -1, "null tensor"), (dict(q=None), -1, "null tensor"), (dict(bt=None), -1, "null tensor"),
    (dict(cl=None), -1, "null tensor"), (dict(kps=None), -1, "null stride"), (dict(B=0), -1, "nonzero"), (dict(D=0), -1, "nonzero"),
    (dict(Hk=3), -1, "multiple"), (dict(Hk=0), -1, "nonzero"), (dict(S=0), -1, "pool dimensions"), (dict(M=0), -1, "block column"),
    (dict(shared=9), -1, "shared_blocks"), (dict(shared=-1), -1, "shared_blocks"), (dict(layer=1), -1, "layer_idx"),
    (dict(dt=4), -1, "dtype"), (dict(bti=3), -1, "int32 or int64"), (dict(cli=3), -1, "int32 or int64"),
    (dict(scale=float("nan")), -1, "scale"), (dict(bts=_st(-8, 1)), -1, "non-negative"), (dict(cls=-1), -1, "non-negative"),
    (dict(B=65536), -2, "65535"), (dict(Hq=70000), -2, "65535"), (dict(B=60000, Hq=600), -2, "too large"),
    (dict(M=1 << 27), -2, "2^30"), (dict(D=513), -2, "512")])
def test_entry_refuses(change, code, msg):
    lib = _native.lib()
    assert lib.mgi_paged_decode_shared(*{**CALL, **change}.values()) == code
    assert msg in lib.mgi_last_error().decode()


def test_workspace_is_asked_for_and_checked(monkeypatch):
    monkeypatch.setenv("MINIVLLM_HIP_SHARED_SPLIT", "1")
    lib = _native.lib()
    size = lib.mgi_paged_decode_shared_workspace_bytes
    n = size(2, 8, 2, 64, 16, 8, 4, 1)
    assert n > 2 * 8 * (64 + 2) * 4
    assert lib.mgi_paged_decode_shared(*CALL.values()) == _native.MGI_EWORKSPACE
    assert lib.mgi_paged_decode_shared(*{**CALL, "ws": P, "bytes": n - 1}.values()) == _native.MGI_EWORKSPACE
    assert lib.mgi_paged_decode_shared(*{**CALL, "ws": ctypes.c_void_p(4104), "bytes": n}.values()) == _native.MGI_EINVAL
    monkeypatch.setenv("MINIVLLM_HIP_SHARED_SPLIT", "0")
    assert size(2, 8, 2, 64, 16, 8, 4, 1) == 0  # one launch needs none
    monkeypatch.delenv("MINIVLLM_HIP_SHARED_SPLIT")
    assert size(2, 8, 2, 20, 16, 8, 4, 1) == 0 and size(2, 8, 2, 512, 16, 8, 4, 1) == 0
    assert size(5000, 8, 2, 64, 16, 8, 4, 1) == 0  # more rows than the split form takes
    assert size(0, 8, 2, 64, 16, 8, 4, 1) == 0 and size(2, 7, 2, 64, 16, 8, 4, 1) == 0


def test_cpu_tensors_are_refused():
    pool = KVBlockPool(1, 4, 16, 2, 64)
    with pytest.raises(ValueError, match="q must be on a GPU device"):
        hpd.paged_attention_shared_prefix_hip(torch.zeros(1, 2, 64), pool, torch.zeros(1, 1, dtype=torch.long),
                                              torch.ones(1, dtype=torch.long), 0, shared_blocks=1)
