"""mgi_prompt_attention without a GPU: its refusals (every one returns before any HIP
call)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from minivllm import _ctypes_ops, _native
from minivllm import hip_paged_decode as hpd

P = ctypes.c_void_p(4096)  # never read: the calls are refused on the host


def _st(*s):
    return (ctypes.c_int64 * len(s))(*s)


CALL = dict(out=P, os=_st(512, 64, 1), q=P, qs=_st(512, 64, 1), k=P, ks=_st(128, 64, 1), v=P, vs=_st(128, 64, 1), dt=1,
            starts=P, ss=1, si=1, B=2, T=50, Hq=8, Hk=2, D=64, scale=0.125, zero=1, stream=None)


@pytest.mark.parametrize("change,code,msg", [
    (dict(out=None), -1, "null tensor"), (dict(q=None), -1, "null tensor"), (dict(k=None), -1, "null tensor"),
    (dict(v=None), -1, "null tensor"), (dict(starts=None), -1, "null tensor"), (dict(os=None), -1, "null stride"),
    (dict(ks=None), -1, "null stride"), (dict(Hq=0), -1, "nonzero"), (dict(D=0), -1, "nonzero"), (dict(Hk=0), -1, "nonzero"),
    (dict(Hk=3), -1, "multiple"), (dict(T=-1), -1, "non-negative"), (dict(B=-1), -1, "non-negative"), (dict(dt=7), -1, "dtype"),
    (dict(si=2), -1, "int32 or int64"), (dict(scale=float("nan")), -1, "scale"), (dict(vs=_st(128, -64, 1)), -1, "non-negative"),
    (dict(ss=-1), -1, "non-negative"), (dict(D=257), -2, "256"), (dict(T=1 << 28), -2, "too large"), (dict(B=1 << 28), -2, "too large"),
    (dict(T=1 << 27, Hq=65536, Hk=65536), -2, "too large"), (dict(T=1 << 27, B=1, Hq=1024), -2, "too large"), (dict(T=0), 0, "")])
def test_entry_refuses(change, code, msg):
    lib = _native.lib()
    assert lib.mgi_prompt_attention(*{**CALL, **change}.values()) == code
    assert msg in lib.mgi_last_error().decode()


@pytest.mark.parametrize("ops", ["extension", "ctypes"])
def test_cpu_tensors_are_refused(ops, monkeypatch):
    if ops == "ctypes":
        monkeypatch.setattr(_native, "_ops", _ctypes_ops)
    x = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="^q must be on a GPU device for the HIP backend$"):
        hpd.prompt_attention_hip(x, x, x, torch.tensor([0, 3]))


@pytest.mark.parametrize("scale", [2.0 ** 127, -3.4e38])
def test_a_scale_whose_exponent_overflows_is_refused(scale):
    lib = _native.lib()
    assert lib.mgi_prompt_attention(*{**CALL, "scale": scale}.values()) == _native.MGI_EUNSUPPORTED
    assert "2^127" in lib.mgi_last_error().decode()
