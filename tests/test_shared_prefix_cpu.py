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


def one_launch(B, Hq, Hk, D, shared, tokens, dtype=1, S=16):
    """Whether a call whose table holds `tokens` takes one launch (no workspace)."""
    return _native.lib().mgi_paged_decode_shared_workspace_bytes(B, Hq, Hk, D, S, -(-tokens // S), shared // S, dtype) == 0


@pytest.mark.parametrize("B,Hq,Hk,D,shared,tokens,dtype", [
    # what each row reads again of the shared tokens: 401 us against 113 with 64 x 32 heads
    (64, 32, 32, 128, 4096, 5120, 1), (64, 32, 8, 128, 4096, 8192, 1), (64, 32, 32, 128, 1024, 4096, 1),
    (32, 32, 8, 128, 2048, 4096, 1), (24, 12, 12, 64, 1504, 1904, 0),
    # one full row among short ones, however wide the table
    (16, 16, 16, 128, 0, 8192, 1), (64, 32, 8, 128, 128, 16384, 2), (256, 32, 32, 128, 0, 4096, 1),
    # rows by the thousand, with few tokens or none: 48 us against 18 and more
    (178, 33, 33, 128, 0, 64, 1), (232, 46, 46, 128, 0, 128, 0)])
def test_wide_tables_keep_the_split(B, Hq, Hk, D, shared, tokens, dtype, monkeypatch):
    for name in ("SPLIT", "LDS"):
        monkeypatch.delenv("MINIVLLM_HIP_SHARED_" + name, raising=False)
    for wider in (1, 2, 4, 16, 64, 256):
        assert not one_launch(B, Hq, Hk, D, shared, shared + (tokens - shared) * wider, dtype), wider


def test_small_calls_take_one_launch(monkeypatch):
    monkeypatch.delenv("MINIVLLM_HIP_SHARED_SPLIT", raising=False)
    for call in ((4, 8, 8, 32, 128, 256, 0), (13, 16, 16, 128, 800, 1312, 1), (1, 8, 2, 128, 0, 512, 2),
                 (8, 8, 8, 64, 64, 512, 1), (32, 8, 8, 128, 16, 256, 1)):
        assert one_launch(*call), call


def test_one_long_row_ends_soon_where_one_launch_is_taken(monkeypatch):
    """Over the ranges calls come in: one workgroup's turns of eight tiles for a full
    row, 1.7 us each 16 KiB, stay below what the split takes for that row and the shared
    tokens, and so does reading the shared tokens by every row, a tenth aside."""
    monkeypatch.delenv("MINIVLLM_HIP_SHARED_SPLIT", raising=False)
    taken = 0
    for dtype, eb, keys in ((1, 2, 32), (0, 4, 16)):
        for Hk in (1, 2, 8, 32):
            for G in (1, 8, 40):
                for D, width in ((32, 64), (64, 64), (128, 128), (256, 256)):
                    for B in (1, 4, 13, 64, 256):
                        for shared in (0, 128, 4096, 65536):
                            for own in (16, 256, 1024, 4096, 16384, 131072):
                                if not one_launch(B, Hk * G, Hk, D, shared, shared + own, dtype):
                                    continue
                                if B * Hk * ((G + 15) // 16) >= 1 << 14 and 2 * B * Hk * G * D * 4 > 4 << 30:
                                    continue  # no partials past 4 GiB
                                taken += 1
                                mb, vheads = 2e-6 * D * eb, Hk * -(-G // 16)
                                mflop = 4e-6 * B * G * Hk * shared * D / (507 if eb == 2 else 63)
                                split = 13 + Hk * shared * mb / 6 + mflop
                                turns = -(-(shared + own) // keys) // 8
                                long = 4.5 + 1.72 * (width * eb / 256) ** 0.73 * turns
                                assert long <= 1.1 * (split + Hk * own * mb / 6), (B, Hk, G, D, shared, own, dtype)
                                assert 4.5 + B * vheads * shared * mb / 10.6 <= 1.1 * split, (B, Hk, G, D, shared, own, dtype)
    assert taken > 300
