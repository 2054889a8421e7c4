"""The rotary calls without a GPU: the table, and the C entries' refusals (every
one returns before any HIP call)."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from minivllm import _native
from minivllm import hip_paged_decode as hpd
from minivllm.kv_block_pool import KVBlockPool


def test_table_holds_cosines_then_sines_of_64_bit_angles():
    t = hpd.rope_table(130000, 8, base=500.0)
    assert t.shape == (130000, 8) and t.dtype == torch.float32
    for p in (0, 1, 77777, 129999):
        for i in range(4):
            a = p * 500.0 ** (-2 * i / 8)
            assert abs(t[p, i].item() - math.cos(a)) <= 2.0 ** -24
            assert abs(t[p, 4 + i].item() - math.sin(a)) <= 2.0 ** -24
    for bad in ((0, 8), (4, 7), (4, 0)):
        with pytest.raises(ValueError, match="rope_table needs"):
            hpd.rope_table(*bad)


def test_cpu_tensors_are_refused():
    q, pos = torch.zeros(2, 4, 64), torch.zeros(2, dtype=torch.long)
    table = hpd.rope_table(4, 64)
    with pytest.raises(ValueError, match="q must be on a GPU device"):
        hpd.qk_norm_rope_hip(q, q, pos, table)
    pool = KVBlockPool(1, 2, 4, 4, 64)
    with pytest.raises(ValueError, match="KV pool must be on a GPU device"):
        hpd.kv_append_rope_hip(pool, 0, q, q, q, pos, pos, table)


P = ctypes.c_void_p(4096)  # never read: the calls are refused on the host


def _st(*s):
    return (ctypes.c_int64 * len(s))(*s)


NORM = dict(qo=P, qos=_st(512, 64, 1), ko=P, kos=_st(128, 64, 1), q=P, qs=_st(512, 64, 1), k=P, ks=_st(128, 64, 1),
            dt=1, pos=P, ps=1, pi=1, tab=P, ts=64, rows=10, R=64, qw=None, kw=None, wd=0, eps=1e-6, inter=0, T=2, Hq=8,
            Hk=2, D=64, stream=None)
APPEND = dict(qo=P, qos=_st(512, 64, 1), kp=P, vp=P, kps=_st(8192, 2048, 128, 64, 1), vps=_st(8192, 2048, 128, 64, 1), pd=1,
              q=P, qs=_st(512, 64, 1), k=P, ks=_st(128, 64, 1), v=P, vs=_st(128, 64, 1), dt=1, sl=P, ss=1, si=1, pos=P,
              ps=1, pi=1, tab=P, ts=64, rows=10, R=64, qw=None, kw=None, wd=0, eps=1e-6, inter=0, T=2, Hq=8, Hk=2, D=64,
              S=16, N=4, L=1, layer=0, stream=None)

SHARED = [(dict(T=-1), -1, "row count"), (dict(qo=None), -1, "null tensor"), (dict(q=None), -1, "null tensor"),
          (dict(pos=None), -1, "null tensor"), (dict(tab=None), -1, "null tensor"), (dict(qs=None), -1, "null stride"),
          (dict(Hq=0), -1, "nonzero"), (dict(Hk=0), -1, "nonzero"), (dict(D=0), -1, "nonzero"), (dict(pi=2), -1, "int32 or int64"),
          (dict(R=63), -1, "rotary_dim"), (dict(R=0), -1, "rotary_dim"), (dict(R=66), -1, "rotary_dim"), (dict(rows=0), -1, "at least one"),
          (dict(qw=P), -1, "come together"), (dict(qw=P, kw=P, wd=2), -1, "norm weights"), (dict(eps=float("inf")), -1, "eps"),
          (dict(eps=-1.0), -1, "eps"), (dict(D=514), -2, "512"), (dict(T=1 << 24), -2, "too large"), (dict(Hq=70000), -2, "too large"),
          (dict(T=1 << 21, Hq=40), -2, "too large"), (dict(ps=-1), -1, "non-negative"), (dict(ts=-64), -1, "non-negative")]


@pytest.mark.parametrize("change,code,msg", SHARED + [
    (dict(ko=None), -1, "null tensor"), (dict(kos=None), -1, "null stride"), (dict(kos=_st(-1, 64, 1)), -1, "non-negative"),
    (dict(dt=7), -1, "dtype")])
def test_norm_rope_entry_refuses(change, code, msg):
    lib = _native.lib()
    assert lib.mgi_qk_norm_rope(*{**NORM, **change}.values()) == code
    assert msg in lib.mgi_last_error().decode()


@pytest.mark.parametrize("change,code,msg", SHARED + [
    (dict(kp=None), -1, "null tensor"), (dict(v=None), -1, "null tensor"), (dict(sl=None), -1, "null tensor"),
    (dict(kps=None), -1, "null stride"), (dict(S=0), -1, "pool dimensions"), (dict(layer=1), -1, "layer_idx"),
    (dict(pd=5), -1, "dtype"), (dict(dt=5), -1, "dtype"), (dict(dt=2), -2, "same-dtype"), (dict(si=5), -1, "slot_mapping"),
    (dict(vps=_st(1, 1, -1, 1, 1)), -1, "non-negative"), (dict(S=1 << 31), -2, "block size")])
def test_append_rope_entry_refuses(change, code, msg):
    lib = _native.lib()
    assert lib.mgi_kv_append_rope(*{**APPEND, **change}.values()) == code
    assert msg in lib.mgi_last_error().decode()


def test_no_rows_is_nothing_to_do():
    lib = _native.lib()
    assert lib.mgi_qk_norm_rope(*{**NORM, "T": 0, "q": None}.values()) == 0
    assert lib.mgi_kv_append_rope(*{**APPEND, "T": 0, "q": None}.values()) == 0
