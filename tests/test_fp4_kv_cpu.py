"""The 4-bit KV pool without a GPU: FP4KVBlockPool's own reads and writes, and the
refusals of mgi_kv_append_fp4, mgi_kv_gather_fp4 and mgi_paged_decode_fp4 (every one
returns before any HIP call)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from minivllm import _ctypes_ops, _native
from minivllm import hip_paged_decode as hpd
from minivllm.kv_block_pool import FP4KVBlockPool
from minivllm.sequence import SequenceState

P = ctypes.c_void_p(4096)  # never read: the calls are refused on the host


def held(row):
    """What a row of D elements is held as, element by element in 64 bits."""
    values = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    out = []
    for g in range(0, len(row), 32):
        group = [float(x) for x in row[g:g + 32]]
        if any(x != x or abs(x) == float("inf") for x in group):
            out += [float("nan")] * len(group)
            continue
        e = -125
        while max(abs(x) for x in group) > 7 * 2.0 ** e and e < 125:
            e += 1
        for x in group:
            y = abs(x) / 2.0 ** e
            best = min(range(8), key=lambda i: (abs(values[i] - y), i % 2))  # ties to the even code
            out.append(values[best] * 2.0 ** e * (-1 if x < 0 else 1))
    return torch.tensor(out, dtype=torch.float64)


SPECIAL = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -7.0, 6.9, 0.0, -0.0,
           0.2500001, 0.7499999, 1.2500001, 1.7499999, 2.5000002, 3.4999998, 5.0000005, 4.0, 6.0, 2.0, 3.0, 1.5, 0.5]


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -124, 2.0 ** 124, 1e-3, 2.0 ** -149 * 64])
def test_ties_and_borders(scale):
    pool = FP4KVBlockPool(1, 1, 1, 1, 32)
    row = (torch.tensor(SPECIAL) * scale).view(1, 1, 32)
    pool.write(0, 0, row, -row)
    seq = SequenceState("s", 1, [0])
    seq.block_table, seq.length = [0], 1
    k, v = pool.gather_sequence(seq)
    assert torch.equal(k.double().flatten(), held(row.flatten()))
    assert torch.equal(v.double().flatten(), held(-row.flatten()))


@pytest.mark.parametrize("D,S", [(1, 1), (7, 5), (32, 16), (80, 16), (128, 16), (160, 3), (256, 8)])
def test_write_and_gather(D, S):
    g = torch.Generator().manual_seed(D)
    pool = FP4KVBlockPool(2, 3, S, 2, D)
    assert pool.data.shape[3] == _native.lib().mgi_fp4_slab_bytes(S, D)
    seq = SequenceState("s", 1, [0])
    seq.block_table, seq.length = [2, 0], 2 * S
    k, v = (torch.randn((2, 2 * S, 2, D), generator=g) * 3 for _ in range(2))
    k[1, 0, 0, 0], v[1, 0, 1, D - 1] = float("nan"), float("inf")
    for t in range(2 * S):
        if t % 2:
            for layer in range(2):
                pool.write_layer(layer, seq.block_table[t // S], t % S, k[layer, t], v[layer, t])
        else:
            pool.write(seq.block_table[t // S], t % S, k[:, t], v[:, t])
    got = pool.gather_sequence(seq)
    for x, y in zip((k, v), got):
        want = torch.stack([held(r) for r in x.reshape(-1, D)]).view(x.shape)
        assert torch.equal(y.double().nan_to_num(nan=-77.0), want.nan_to_num(nan=-77.0))


def test_pool_refuses():
    with pytest.raises(ValueError, match="head_dim"):
        FP4KVBlockPool(1, 1, 16, 1, 257)
    with pytest.raises(ValueError, match="head_dim"):
        FP4KVBlockPool(1, 1, 16, 1, 0)
    with pytest.raises(ValueError, match="block_size"):
        FP4KVBlockPool(1, 1, 0, 1, 64)
    size = _native.lib().mgi_fp4_slab_bytes
    assert size(16, 128) == 16 * 4 * 34 and size(1, 1) == 48
    assert size(0, 64) == size(16, 0) == size(16, 257) == size((1 << 20) + 1, 64) == 0


def _st(*s):
    return (ctypes.c_int64 * len(s))(*s)


ROWS = dict(slots=P, ss=1, si=1, T=2, H=2, D=64, S=16, N=4, L=1, layer=0, stream=None)
APPEND = dict(pool=P, ps=_st(8704, 2176, 1088), k=P, v=P, ks=_st(128, 64, 1), vs=_st(128, 64, 1), dt=1, **ROWS)
GATHER = dict(k=P, v=P, ks=_st(128, 64, 1), vs=_st(128, 64, 1), dt=1, pool=P, ps=_st(8704, 2176, 1088), **ROWS)


@pytest.mark.parametrize("change,code,msg", [
    (dict(pool=None), -1, "null tensor"), (dict(ps=None), -1, "null stride"), (dict(k=None), -1, "null tensor"),
    (dict(v=None), -1, "null tensor"), (dict(slots=None), -1, "null tensor"), (dict(ks=None), -1, "null stride"),
    (dict(dt=3), -1, "dtype"), (dict(si=2), -1, "int32 or int64"), (dict(T=-1), -1, "non-negative"),
    (dict(H=0), -1, "nonzero"), (dict(D=0), -1, "nonzero"), (dict(S=0), -1, "nonzero"), (dict(N=0), -1, "nonzero"),
    (dict(layer=1), -1, "layer_idx"), (dict(layer=-1), -1, "layer_idx"), (dict(ps=_st(8704, 2176, 1080)), -1, "aligned"),
    (dict(pool=ctypes.c_void_p(4104)), -1, "aligned"), (dict(ps=_st(-16, 2176, 1088)), -1, "non-negative"),
    (dict(ks=_st(-1, 64, 1)), -1, "non-negative"), (dict(ss=-1), -1, "non-negative"),
    (dict(D=257), -2, "256"), (dict(H=65536), -2, "65535"), (dict(S=(1 << 20) + 1), -2, "block size"),
    (dict(N=1 << 31), -2, "blocks"), (dict(T=1 << 24), -2, "rows"), (dict(H=65535, D=256, T=1 << 20), 0, "")])
def test_rows_refuse(change, code, msg):
    lib = _native.lib()
    if code == 0:  # inside the limits: only that the limits meet (nothing is launched with no rows)
        change = {**change, "T": 0}
    for call, base in ((lib.mgi_kv_append_fp4, APPEND), (lib.mgi_kv_gather_fp4, GATHER)):
        assert call(*{**base, **change}.values()) == code
        assert msg in lib.mgi_last_error().decode()


DECODE = dict(out=P, os=_st(512, 64, 1), q=P, qs=_st(512, 64, 1), dt=1, pool=P, ps=_st(8704, 2176, 1088), bt=P,
              bts=_st(8, 1), bti=1, cl=P, cls=1, cli=1, B=2, Hq=8, Hk=2, D=64, S=16, N=4, M=8, L=1, layer=0, scale=0.125,
              ws=None, bytes=0, stream=None)


@pytest.mark.parametrize("change,code,msg", [
    (dict(out=None), -1, "null tensor"), (dict(q=None), -1, "null tensor"), (dict(bt=None), -1, "null tensor"),
    (dict(cl=None), -1, "null tensor"), (dict(pool=None), -1, "null tensor"), (dict(qs=None), -1, "null stride"),
    (dict(ps=None), -1, "null stride"), (dict(B=0), -1, "nonzero"), (dict(D=0), -1, "nonzero"), (dict(Hk=3), -1, "multiple"),
    (dict(Hk=0), -1, "nonzero"), (dict(S=0), -1, "nonzero"), (dict(M=0), -1, "block column"), (dict(layer=1), -1, "layer_idx"),
    (dict(dt=4), -1, "dtype"), (dict(bti=3), -1, "int32 or int64"), (dict(cli=3), -1, "int32 or int64"),
    (dict(scale=float("inf")), -1, "scale"), (dict(bts=_st(-8, 1)), -1, "non-negative"), (dict(cls=-1), -1, "non-negative"),
    (dict(ps=_st(8704, 2176, 1089)), -1, "aligned"), (dict(B=65536), -2, "65535"), (dict(Hq=70000), -2, "65535"),
    (dict(B=60000, Hq=600), -2, "too large"), (dict(M=1 << 27), -2, "2^30"), (dict(B=60000, M=1 << 20), -2, "2^35"),
    (dict(D=257), -2, "256")])
def test_decode_refuses(change, code, msg):
    lib = _native.lib()
    assert lib.mgi_paged_decode_fp4(*{**DECODE, **change}.values()) == code
    assert msg in lib.mgi_last_error().decode()


def test_workspace_is_asked_for_and_checked(monkeypatch):
    lib = _native.lib()
    size = lib.mgi_paged_decode_fp4_workspace_bytes
    monkeypatch.setenv("MINIVLLM_HIP_FP4_SPLIT", "1")
    n = size(2, 8, 2, 64, 16, 8)
    assert n > 2 * 8 * (64 + 2) * 4
    assert lib.mgi_paged_decode_fp4(*DECODE.values()) == _native.MGI_EWORKSPACE
    assert lib.mgi_paged_decode_fp4(*{**DECODE, "ws": P, "bytes": n - 1}.values()) == _native.MGI_EWORKSPACE
    assert lib.mgi_paged_decode_fp4(*{**DECODE, "ws": ctypes.c_void_p(4104), "bytes": n}.values()) == _native.MGI_EINVAL
    monkeypatch.setenv("MINIVLLM_HIP_FP4_SPLIT", "0")
    assert size(2, 8, 2, 64, 16, 8) == 0
    monkeypatch.delenv("MINIVLLM_HIP_FP4_SPLIT")
    assert size(0, 8, 2, 64, 16, 8) == size(2, 7, 2, 64, 16, 8) == size(2, 8, 2, 257, 16, 8) == 0
    assert size(64, 32, 32, 128, 16, 8192) > 0


@pytest.mark.parametrize("ops", ["extension", "ctypes"])
def test_cpu_tensors_are_refused(ops, monkeypatch):
    if ops == "ctypes":
        monkeypatch.setattr(_native, "_ops", _ctypes_ops)
    pool = FP4KVBlockPool(1, 4, 16, 2, 64)
    rows, ids = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.long)
    with pytest.raises(ValueError, match="^KV pool must be on a GPU device for the HIP backend$"):
        hpd.kv_append_fp4(pool, 0, rows, rows, ids)
    with pytest.raises(ValueError, match="^KV pool must be on a GPU device for the HIP backend$"):
        hpd.kv_gather_fp4(pool, 0, ids)
    with pytest.raises(ValueError, match="^q must be on a GPU device for the HIP backend$"):
        hpd.paged_attention_fp4_hip(rows, pool, ids[:, None], ids, 0)


@pytest.mark.parametrize("scale", [2.0 ** 127, -3.4e38])
def test_a_scale_whose_exponent_overflows_is_refused(scale):
    lib = _native.lib()
    assert lib.mgi_paged_decode_fp4(*{**DECODE, "scale": scale}.values()) == _native.MGI_EUNSUPPORTED
    assert "2^127" in lib.mgi_last_error().decode()


def test_one_launch_or_two_by_the_wavefronts_a_call_has(monkeypatch):
    """At most 8 tiles of 32 tokens for a wavefront in one launch; f32 heads of more than 192
    dims have 4 wavefronts to a workgroup, other calls 8."""
    lib = _native.lib()
    monkeypatch.delenv("MINIVLLM_HIP_FP4_SPLIT", raising=False)
    size = lib.mgi_paged_decode_fp4_workspace_bytes
    for D in (193, 256):  # 1024 tokens, and 1040
        slab = lib.mgi_fp4_slab_bytes(16, D)
        call = {**DECODE, "D": D, "dt": 0, "Hq": 2, "ps": _st(4 * 2 * slab, 2 * slab, slab), "M": 65}
        assert lib.mgi_paged_decode_fp4(*call.values()) == _native.MGI_EWORKSPACE
        assert size(2, 2, 2, D, 16, 64) == 0 and size(2, 2, 2, D, 16, 65) > 0
    for D in (64, 192):
        assert size(2, 2, 2, D, 16, 128) == 0 and size(2, 2, 2, D, 16, 129) > 0
    # Partials of the wavefronts that are resident: two for each of 2 per SIMD, 256 dims, 16 rows.
    assert size(64, 128, 8, 256, 16, 8192) <= 1.05 * 2 * (8 * 256) * 16 * (256 + 2) * 4
