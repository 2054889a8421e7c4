"""The 4-bit KV pool's kernels: kv_append_fp4 and kv_gather_fp4 byte by byte against
FP4KVBlockPool's own reads and writes (checked element by element in
test_fp4_kv_cpu.py), paged_attention_fp4_hip against the softmax in 64 bits over the
values that the pool holds.

Tolerance of the attention. With A = sum_t w_t |V_t| (w the softmax weights), u = 2^-24
and n keys:
 - a score is a sum of D exact products in f32: off by at most D u X, X = scale sum_d
   |q_d k_d|; scaling, the exponent's difference and exp2 add 4 u (1 + X); a weight and
   the sum that divides it are each off by that: 2 (D + 4) u max_t X + 8 u;
 - n additions into output and sum, joined over pieces: 2 (n + 32) u;
 - a weight is cut into two bf16 terms, each rounded by half a step: 2^-18 of the weight
   (f32: three terms, 2^-27), for the output alone: 2^-18 of A;
 - the output's rounding: eps / 2 of itself (f32: u)."""
from __future__ import annotations

import math

import pytest
import torch

from minivllm import _ctypes_ops, _native
from minivllm import hip_paged_decode as hpd
from minivllm.kv_block_pool import FP4KVBlockPool

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
ROUTES = pytest.mark.parametrize("route", ["one", "split"])


@pytest.fixture(autouse=True)
def _route(request, monkeypatch):
    route = request.node.callspec.params.get("route") if hasattr(request.node, "callspec") else None
    if route:
        monkeypatch.setenv("MINIVLLM_HIP_FP4_SPLIT", "0" if route == "one" else "1")


def cpu_pool(L, N, S, H, D):
    pool = FP4KVBlockPool(L, N, S, H, D)
    pool.data.fill_(255)
    return pool


def gpu_pool(host):
    pool = FP4KVBlockPool(host.n_layer, host.num_blocks, host.block_size, host.n_head, host.head_dim, device=DEV)
    pool.data.copy_(host.data)
    return pool


# ------------------------------------------------------------ append, gather

@DTYPES
@pytest.mark.parametrize("T,H,D,S,itype,strided", [
    (1, 1, 1, 1, torch.int64, False), (5, 2, 7, 5, torch.int32, False), (4, 8, 32, 16, torch.int64, True),
    (33, 3, 80, 16, torch.int64, True), (64, 2, 128, 8, torch.int32, True), (17, 1, 160, 3, torch.int64, False),
    (9, 2, 256, 16, torch.int64, True), (70, 5, 96, 32, torch.int64, True), (600, 2, 20, 7, torch.int64, False)])
def test_append_is_the_pools_own_write(T, H, D, S, itype, strided, dtype):
    g = torch.Generator().manual_seed(T + D)
    N, layer = T // S + 3, 1
    host = cpu_pool(2, N, S, H, D)
    pool = gpu_pool(host)
    rows = (torch.randn((T, 3 * H, D), generator=g) * torch.exp(2 * torch.randn((T, 3 * H, 1), generator=g))).to(dtype)
    k, v = rows[:, H:2 * H], rows[:, 2 * H:]
    if T > 8:  # groups that hold what is not a number, zeros, one sign
        k[1, 0, D // 2], v[2, H - 1, 0] = float("nan"), float("-inf")
        k[3], v[4], k[5] = 0, -0.0, k[5].abs() * -1
    slots = torch.randperm(N * S, generator=g)[:T]
    slots[T // 2] = -1 if T > 2 else slots[T // 2]
    if T > 4:
        slots[T // 3] = N * S + 5
    dk, dv = (k.to(DEV), v.to(DEV)) if not strided else (rows.to(DEV)[:, H:2 * H], rows.to(DEV)[:, 2 * H:])
    hpd.kv_append_fp4(pool, layer, dk, dv, slots.to(itype).to(DEV))
    for t in range(T):
        s = int(slots[t])
        if 0 <= s < N * S:
            host.write_layer(layer, s // S, s % S, k[t], v[t])
    assert torch.equal(pool.data.cpu(), host.data)
    # Reading back: every slot the pool has, and some it has not.
    ids = torch.cat((torch.arange(N * S), torch.tensor([-1, N * S, -(1 << 40) if itype == torch.int64 else -7])))
    got = hpd.kv_gather_fp4(pool, layer, ids.to(itype).to(DEV), dtype=dtype)
    parts = host._parts(host.data[layer])
    for x, codes, scales in zip(got, parts[:2], parts[2:]):
        want = host._decode(codes, scales, dtype).transpose(1, 2).reshape(N * S, H, D)
        assert x.shape == (N * S + 3, H, D) and x.dtype == dtype
        assert torch.equal(x[:N * S].cpu().float().nan_to_num(nan=-77.0), want.float().nan_to_num(nan=-77.0))
        assert (x[N * S:] == 0).all()


@DTYPES
def test_ties_borders_and_extremes(dtype):
    """Every border between codes and its neighbours, at scales over the whole range."""
    y = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 4.0, 3.0, 2.0, 1.5, 1.0, 0.5, 0.0])
    eps = torch.finfo(dtype).eps
    rows = []
    for top in (7.0, 6.0, 4.0, 3.5, 7.0 * (1 - eps), 7.0 * (1 + eps), 3.5 * (1 + eps)):
        for near in (1 - eps, 1.0, 1 + eps):
            group = (y * near).clamp(max=top)
            group[0] = top
            rows.append(torch.cat((group, -group)))
    rows = torch.stack(rows)  # [21, 32]
    lo, hi = (-20, 12) if dtype == F16 else (-126, 124)
    x = torch.cat([rows * 2.0 ** e for e in (lo, lo + 1, lo + 9, -3, 0, 5, hi)]).to(dtype)[:, None]  # [T, 1, 32]
    x = torch.cat((x, torch.full_like(x[:1], 2.0 ** -149 if dtype == F32 else torch.finfo(dtype).tiny), torch.zeros_like(x[:1])))
    T = len(x)
    host = cpu_pool(1, T, 1, 1, 32)
    pool = gpu_pool(host)
    hpd.kv_append_fp4(pool, 0, x.to(DEV), -x.to(DEV), torch.arange(T, device=DEV))
    for t in range(T):
        host.write_layer(0, t, 0, x[t], -x[t])
    assert torch.equal(pool.data.cpu(), host.data)


def test_append_takes_any_strides():
    g = torch.Generator().manual_seed(3)
    T, H, D, S = 13, 3, 48, 16
    k, v = torch.randn((2, D, H, T), generator=g).to(DEV)
    k, v = k.permute(2, 1, 0), v.permute(2, 1, 0)
    slots = torch.arange(2 * T, device=DEV)[::2] + 3
    host = cpu_pool(1, 4, S, H, D)
    pool, twin = gpu_pool(host), gpu_pool(host)
    hpd.kv_append_fp4(pool, 0, k, v, slots)
    hpd.kv_append_fp4(twin, 0, k.contiguous(), v.contiguous(), slots.contiguous())
    assert torch.equal(pool.data, twin.data) and not torch.equal(pool.data.cpu(), host.data)


@pytest.mark.parametrize("T", [2, 40, 257, 1500, 6000, 70000])
def test_of_rows_on_one_slot_the_last_is_kept_whole(T):
    g = torch.Generator().manual_seed(T)
    H, D, S, N = 2, 64, 16, 8 if T < 10000 else T // 16
    k, v = (torch.randn((2, T, H, D), generator=g) * torch.exp(3 * torch.randn((2, T, 1, 1), generator=g))).to(DEV)
    slots = torch.randint(-1, N * S, (T,), generator=g)
    slots[0] = slots[T - 1]
    last = {int(s): t for t, s in enumerate(slots) if s >= 0}
    pool, twin = (gpu_pool(cpu_pool(1, N, S, H, D)) for _ in range(2))
    hpd.kv_append_fp4(pool, 0, k, v, slots.to(DEV))
    rows = torch.tensor(list(last.values()), device=DEV)
    hpd.kv_append_fp4(twin, 0, k[rows], v[rows], torch.tensor(list(last), device=DEV))
    assert torch.equal(pool.data, twin.data)


def test_values_outside_float16_come_out_infinite():
    pool = gpu_pool(cpu_pool(1, 1, 16, 1, 32))
    x = torch.full((1, 1, 32), 3.0e38, device=DEV)
    x[0, 0, 0] = 3.4e38
    hpd.kv_append_fp4(pool, 0, x, -x, torch.zeros(1, dtype=torch.long, device=DEV))
    k, v = hpd.kv_gather_fp4(pool, 0, torch.zeros(1, dtype=torch.long, device=DEV))
    assert (k == 6 * 2.0 ** 125).all() and (v == -6 * 2.0 ** 125).all()  # the largest that is held
    k, v = hpd.kv_gather_fp4(pool, 0, torch.zeros(1, dtype=torch.long, device=DEV), dtype=F16)
    assert (k == float("inf")).all() and (v == -float("inf")).all()


# ----------------------------------------------------------------- attention

def make(B, Hq, Hk, D, S, ctx, dtype, seed=0, M=None, itype=torch.int64, layer=1):
    """q, pool, tables, lengths; every slot that no row holds is NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(0, c) // S) for c in ctx]
    M = max(1, max(need)) if M is None else M
    N = sum(need) + 2
    perm = torch.randperm(N, generator=g)
    tables = torch.full((B, M), -1, dtype=torch.int64)
    host = cpu_pool(2, N, S, Hk, D)
    parts = host._parts(host.data[layer])
    at = 0
    for b, c in enumerate(ctx):
        if c <= 0:
            continue
        ids = perm[at:at + need[b]]
        at += need[b]
        tables[b, :need[b]] = ids
        for i, (codes, scales) in enumerate((parts[0::2], parts[1::2])):
            x = torch.randn((need[b] * S, Hk, D), generator=g)
            cs, ss = host._encode(x if i else x * torch.exp(0.5 * torch.randn((1, Hk, D), generator=g)))
            for dst, src in ((codes, cs), (scales, ss)):
                src = src.view(need[b], S, Hk, -1)
                left = c - (need[b] - 1) * S
                dst[ids[:-1]] = src[:-1].transpose(1, 2)
                dst[ids[-1], :, :left] = src[-1, :left].transpose(0, 1)
    q = torch.randn((B, Hq, D), generator=g).to(dtype).to(DEV)
    return q, gpu_pool(host), tables.to(itype).to(DEV), torch.tensor(ctx, dtype=itype, device=DEV), layer


def reference(q, pool, tables, ctx, layer, scale=None):
    """(out, A, X, n) in 64 bits; a row without keys gives 0."""
    B, Hq, D = q.shape
    S, Hk, N, M = pool.block_size, pool.n_head, pool.num_blocks, tables.shape[1]
    G = Hq // Hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    kc, vc, ks, vs = pool._parts(pool.data[layer])
    k, v = (pool._decode(c, s, F32).double() for c, s in ((kc, ks), (vc, vs)))  # [N, H, S, D]
    out = torch.zeros((B, Hq, D), dtype=torch.float64, device=DEV)
    A, X, most = torch.zeros_like(out), torch.zeros((B, Hq, 1), dtype=torch.float64, device=DEV), 0
    for b in range(B):
        c = min(max(int(ctx[b]), 0), M * S)
        t = torch.arange(c, device=DEV)
        blk = tables[b, t // S].long()
        ok = (blk >= 0) & (blk < N)
        t, blk = t[ok], blk[ok]
        most = max(most, len(t))
        if len(t) == 0:
            continue
        kb, vb = (x[blk, :, t % S].transpose(0, 1).contiguous() for x in (k, v))  # [H, n, D]
        qb = q[b].double().view(Hk, G, D) * scale
        s = qb @ kb.transpose(1, 2).contiguous()
        w = torch.softmax(s, -1)
        out[b] = (w @ vb).view(Hq, D)
        A[b] = (w @ vb.abs()).view(Hq, D)
        X[b] = (qb.abs() @ kb.abs().transpose(1, 2).contiguous()).amax(-1).view(Hq, 1)
    return out, A, X, most


def check(got, q, pool, tables, ctx, layer, scale=None):
    out, A, X, n = reference(q, pool, tables, ctx, layer, scale)
    D, half = q.shape[2], torch.finfo(q.dtype).eps / 2
    cut = 2.0 ** -27 if q.dtype == F32 else 2.0 ** -18
    tol = (2 * (D + 4) * U * X + 8 * U + 2 * (n + 32) * U + cut) * A + half * out.abs() + 2.0 ** -25 * (q.dtype == F16)
    off = (got.double() - out).abs()
    assert got.shape == q.shape and got.dtype == q.dtype
    assert not torch.isnan(got).any()
    assert (off <= tol).all(), f"worst {float((off / tol.clamp_min(1e-300)).max()):.3g} of the tolerance"


LENGTHS = [1, 0, 31, 32, 33, 200, 64, 1000]


@DTYPES
@ROUTES
@pytest.mark.parametrize("Hq,Hk,D,S", [
    (8, 8, 32, 16), (4, 2, 64, 16), (3, 1, 80, 32), (6, 2, 96, 16), (4, 4, 128, 16), (16, 2, 128, 64), (17, 1, 128, 16),
    (40, 1, 64, 16), (4, 2, 160, 16), (2, 1, 192, 16), (2, 2, 224, 16), (5, 1, 256, 32), (2, 2, 20, 16), (1, 1, 1, 16)])
def test_attention(Hq, Hk, D, S, route, dtype):
    case = make(len(LENGTHS), Hq, Hk, D, S, LENGTHS, dtype, seed=D + Hq)
    check(hpd.paged_attention_fp4_hip(*case), *case)


@DTYPES
@ROUTES
@pytest.mark.parametrize("Hq,Hk,D,S", [(4, 2, 64, 1), (4, 4, 128, 5), (8, 1, 96, 8), (2, 1, 256, 24), (3, 3, 33, 7),
                                       (5, 5, 224, 6), (18, 1, 160, 12), (4, 2, 192, 20)])
def test_block_sizes_that_are_no_multiple_of_16(Hq, Hk, D, S, route, dtype):
    lens = [1, 0, 31, 70, 33, 200]
    case = make(len(lens), Hq, Hk, D, S, lens, dtype, seed=S)
    check(hpd.paged_attention_fp4_hip(*case), *case)


@DTYPES
@pytest.mark.parametrize("Hq,Hk,D,S", [(2, 1, 128, 16), (3, 1, 96, 32), (1, 1, 20, 16), (17, 1, 64, 6)])
def test_few_long_sequences(Hq, Hk, D, S, dtype):
    """Many runs to join for one head."""
    lens = [9001, 1, 0, 4100]
    case = make(len(lens), Hq, Hk, D, S, lens, dtype, seed=D)
    check(hpd.paged_attention_fp4_hip(*case), *case)


@ROUTES
@pytest.mark.parametrize("S", [16, 6])
def test_blocks_outside_the_pool_are_masked(S, route):
    q, pool, tables, ctx, layer = make(4, 8, 4, 64, S, [100, 300, 17, 90], BF16, itype=torch.int32)
    tables[0, 2], tables[1, 0], tables[1, 3] = -1, pool.num_blocks, -(1 << 31)
    tables[2, :] = -1  # no key is left: 0
    got = hpd.paged_attention_fp4_hip(q, pool, tables, ctx, layer)
    check(got, q, pool, tables, ctx, layer)
    assert (got[2] == 0).all()


@ROUTES
def test_lengths_outside_the_table_are_clamped(route):
    q, pool, tables, ctx, layer = make(3, 4, 4, 128, 16, [64, 64, 64], BF16, M=4)
    ctx[0], ctx[1] = 1 << 40, -5
    got = hpd.paged_attention_fp4_hip(q, pool, tables, ctx, layer)
    check(got, q, pool, tables, ctx, layer)
    assert (got[1] == 0).all()


@ROUTES
def test_nan_in_the_context_stays_in_its_row_and_head(route):
    q, pool, tables, ctx, layer = make(3, 4, 2, 64, 16, [50, 50, 50], F32)
    k, v, ks, vs = pool._parts(pool.data[layer])
    ks[tables[0, 1], 0, 3, 1] = 255           # a key group of row 0, KV head 0
    vs[tables[1, 2], 1, 5, 0] = 255           # a value group of row 1, KV head 1: dims 0 .. 31
    got = hpd.paged_attention_fp4_hip(q, pool, tables, ctx, layer)
    lost = torch.isnan(got)
    assert lost[0, :2].all() and not lost[0, 2:].any() and not lost[2].any()
    assert lost[1, 2:, :32].all() and not lost[1, 2:, 32:].any() and not lost[1, :2].any()


@DTYPES
@ROUTES
def test_large_scores_and_far_scales(route, dtype):
    q, pool, tables, ctx, layer = make(2, 4, 2, 64, 16, [300, 77], dtype)
    check(hpd.paged_attention_fp4_hip(q * 60, pool, tables, ctx, layer), q * 60, pool, tables, ctx, layer)
    _, _, ks, vs = pool._parts(pool.data[layer])
    for x, by in ((ks, -60), (vs, 90)):  # keys near 2^-60, values near 2^90
        x.copy_(torch.where(x == 255, 255, x.int() + by).to(torch.uint8))
    if dtype != F16:
        check(hpd.paged_attention_fp4_hip(q, pool, tables, ctx, layer), q, pool, tables, ctx, layer)


def entry(q, pool, tables, ctx, layer, scale, out):
    """The C entry, for what the Python call fixes: the scale, the output's strides."""
    lib = _native.lib()
    B, Hq, D = q.shape
    L, N, H = pool.data.shape[:3]
    n = lib.mgi_paged_decode_fp4_workspace_bytes(B, Hq, H, D, pool.block_size, tables.shape[1])
    ws = torch.empty(max(1, n), dtype=torch.uint8, device=DEV)
    _native.check(lib.mgi_paged_decode_fp4(
        out.data_ptr(), _native.strides(out), q.data_ptr(), _native.strides(q), _native.DTYPE_CODES[q.dtype],
        pool.data.data_ptr(), _native.strides(pool.data), tables.data_ptr(), _native.strides(tables),
        _native.ITYPE_CODES[tables.dtype], ctx.data_ptr(), ctx.stride(0), _native.ITYPE_CODES[ctx.dtype], B, Hq, H, D,
        pool.block_size, N, tables.shape[1], L, layer, scale, ws.data_ptr(), n, _native.stream_handle(DEV)))
    return out


@ROUTES
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-30])
def test_any_scale_and_strides(scale, route):
    q, pool, tables, ctx, layer = make(3, 6, 2, 96, 16, [130, 40, 1], F32)
    strange = q.transpose(0, 2).contiguous().transpose(0, 2)
    wide = torch.full((4, 8, 200), 7.0, device=DEV)
    out = wide[:3, 1:7, 3:195:2]
    entry(strange, pool, tables[:, :, None].expand(-1, -1, 3).contiguous()[:, :, 1], ctx, layer, scale, out)
    check(out, q, pool, tables, ctx, layer, scale)
    assert (wide[3] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, 7] == 7).all() and (wide[..., :3] == 7).all() \
        and (wide[..., 4::2] == 7).all() and (wide[..., 195:] == 7).all()


def test_large_batches_and_uneven_lengths():
    lens = [(i * 37) % 97 if i % 5 else 0 for i in range(300)]
    lens[150] = 5000
    case = make(300, 4, 2, 64, 16, lens, BF16, seed=5)
    assert _native.lib().mgi_paged_decode_fp4_workspace_bytes(300, 4, 2, 64, 16, case[2].shape[1]) > 0
    check(hpd.paged_attention_fp4_hip(*case), *case)


def test_more_rows_than_wavefronts():
    lens = [i % 3 for i in range(3000)]
    case = make(3000, 4, 2, 32, 16, lens, F16, seed=6, M=40)
    check(hpd.paged_attention_fp4_hip(*case), *case)


@ROUTES
def test_same_inputs_same_bits_and_ctypes(route):
    case = make(6, 8, 2, 128, 16, [500, 1, 0, 90, 1200, 33], BF16)
    q, pool, tables, ctx, layer = case
    first = hpd.paged_attention_fp4_hip(*case)
    for _ in range(5):
        assert torch.equal(first, hpd.paged_attention_fp4_hip(*case))
    other = _ctypes_ops.paged_decode_fp4(q, pool.data, 16, 128, tables, ctx, layer)
    assert torch.equal(first, other)
    k = torch.randn((6, 2, 128), device=DEV)
    twin = FP4KVBlockPool(2, pool.num_blocks, 16, 2, 128, device=DEV)
    twin.data.copy_(pool.data)
    slots = torch.tensor([3, -1, 16, 17, 3, 90], device=DEV)
    hpd.kv_append_fp4(pool, 0, k, -k, slots)
    _ctypes_ops.kv_append_fp4(twin.data, 16, 128, 0, k, -k, slots)
    assert torch.equal(pool.data, twin.data)
    for a, b in zip(hpd.kv_gather_fp4(pool, 0, slots, dtype=BF16), _ctypes_ops.kv_gather_fp4(twin.data, 16, 128, 0, slots, BF16)):
        assert torch.equal(a, b) and a.dtype == b.dtype == BF16


def test_offsets_past_32_bits():
    """A pool of more than 4 GiB, its last blocks used."""
    S, H, D, N = 16, 8, 128, 260_000
    pool = FP4KVBlockPool(1, N, S, H, D, device=DEV)
    assert pool.data.numel() > 1 << 32
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn((2, 70, H, D), generator=g).to(BF16).to(DEV)
    tables = torch.tensor([[N - 1, N - 3, 5, N - 7, N - 2]], device=DEV)
    t = torch.arange(70, device=DEV)
    slots = tables[0, t // S] * S + t % S
    hpd.kv_append_fp4(pool, 0, k, v, slots)
    small = FP4KVBlockPool(1, 5, S, H, D, device=DEV)
    hpd.kv_append_fp4(small, 0, k, v, t)
    for a, b in zip(hpd.kv_gather_fp4(pool, 0, slots), hpd.kv_gather_fp4(small, 0, t)):
        assert torch.equal(a, b)
    q, ctx = torch.randn((1, 16, D), generator=g).to(BF16).to(DEV), torch.tensor([70], device=DEV)
    a = hpd.paged_attention_fp4_hip(q, pool, tables, ctx, 0)
    b = hpd.paged_attention_fp4_hip(q, small, torch.arange(5, device=DEV)[None], ctx, 0)
    assert torch.equal(a, b)


@ROUTES
def test_graph_replays_follow_their_inputs(route):
    q, pool, tables, ctx, layer = make(4, 8, 4, 128, 16, [700, 40, 90, 3], BF16)
    k, v = torch.randn((2, 4, 4, 128), device=DEV).to(BF16)
    last = ctx - 1
    slots = tables[torch.arange(4, device=DEV), last // 16] * 16 + last % 16

    def step():
        hpd.kv_append_fp4(pool, layer, k, v, slots)
        return hpd.paged_attention_fp4_hip(q, pool, tables, ctx, layer)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(second, pool=graph.pool()):  # shares the first one's memory
        out2 = step()
    for i in range(4):
        ctx.copy_(torch.tensor([700 - 90 * i, 40, 90 - i, i], device=DEV))
        q.normal_()
        k.normal_()
        graph.replay()
        a = out.clone()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(a, want)
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(out2, want)


@ROUTES
def test_calls_on_two_streams_at_once(route):
    cases = [make(8, 8, 2, 64, 16, [900 - 50 * i for i in range(8)], BF16, seed=s) for s in (1, 2)]
    want = [hpd.paged_attention_fp4_hip(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(hpd.paged_attention_fp4_hip(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    q, pool, tables, ctx, layer = make(2, 4, 2, 64, 16, [20, 30], BF16)
    rows, ids = torch.zeros((2, 2, 64), dtype=BF16, device=DEV), torch.zeros(2, dtype=torch.long, device=DEV)
    for ops in (_native.ops(), _ctypes_ops):
        append = lambda *a: ops.kv_append_fp4(pool.data, 16, 64, *a)
        for args, msg in [((2, rows, rows, ids), "layer_idx"), ((0, rows, rows[:1], ids), "matching shape"),
                          ((0, rows[:, :1], rows[:, :1], ids), "head dimensions"), ((0, rows.double(), rows.double(), ids), "float dtype"),
                          ((0, rows, rows.float(), ids), "float dtype"), ((0, rows, rows, ids[:1]), "slot_mapping"),
                          ((0, rows, rows, ids.float()), "integer"), ((0, rows, rows, ids.cpu()), "same GPU device")]:
            with pytest.raises(ValueError, match=msg):
                append(*args)
        with pytest.raises(RuntimeError, match="inference-only"):
            append(0, rows.clone().requires_grad_(), rows, ids)
        for args, msg in [((pool.data, 32, 64, 0, ids, F32), "slab"), ((pool.data, 16, 300, 0, ids, F32), "head_dim"),
                          ((pool.data, 0, 64, 0, ids, F32), "block_size"), ((pool.data[..., ::2], 16, 64, 0, ids, F32), "slab"),
                          ((pool.data.short(), 16, 64, 0, ids, F32), "uint8"), ((pool.data, 16, 64, 0, ids[None], F32), "slot_mapping"),
                          ((pool.data, 16, 64, 0, ids, torch.float64), "dtype must be")]:
            with pytest.raises(ValueError, match=msg):
                ops.kv_gather_fp4(*args)
        attend = lambda q, bt, cl, layer=0: ops.paged_decode_fp4(q, pool.data, 16, 64, bt, cl, layer)
        for args, msg in [((q[:, :3], tables, ctx), "multiple"), ((q[..., :32], tables, ctx), "head dimension"),
                          ((q.double(), tables, ctx), "float32"), ((q, tables[:1], ctx), r"\[B,M\]"), ((q, tables, ctx[:1]), r"\[B\]"),
                          ((q, tables.float(), ctx), "integer"), ((q, tables, ctx.float()), "integer"), ((q, tables, ctx, 2), "layer_idx"),
                          ((q, tables[:, :0], ctx), "block column"), ((q, tables.cpu(), ctx), "same GPU device"), ((q[0], tables, ctx), "shape")]:
            with pytest.raises(ValueError, match=msg):
                attend(*args)
        with pytest.raises(RuntimeError, match="inference-only"):
            attend(q.clone().requires_grad_(), tables, ctx)
        # Nothing to do.
        append(0, rows[:0], rows[:0], ids[:0])
        assert ops.kv_gather_fp4(pool.data, 16, 64, 0, ids[:0], F32)[0].shape == (0, 2, 64)


@DTYPES
@ROUTES
@pytest.mark.parametrize("S", [16, 6])
@pytest.mark.parametrize("power", [4, 16, 20, 24, 30, 32, 34, 40, 60])
def test_scores_of_any_size(power, S, route, dtype):
    """Scores near 2^power (of e), or a few units (a third of the rows), every one a sum of two products that
    f32 holds exactly: what is left is 3 u of a weight's exponent (the scale's factor, its
    product), which moves a weight 2^-d by 3 u d 2^-d <= 2 u, exp2 and the sums. Weights below
    2^-118 of the largest may be 0 in f32 (its least normal number is 2^-126, and the
    running maximum is up to 2^8 off): n 2^-118 max |v|, which counts where every larger
    weight meets a value of 0."""
    lens = [1, 2, 33, 300, 290, 700]
    g = torch.Generator().manual_seed(power)
    B, H, D, n = len(lens), 2, 64, [-(-c // S) for c in lens]
    pool = gpu_pool(cpu_pool(1, sum(n), S, H, D))
    tables = torch.full((B, max(n)), -1, dtype=torch.int64)
    at = 0
    for b in range(B):
        tables[b, :n[b]] = torch.arange(at, at + n[b])
        at += n[b]
    rows = sum(n) * S
    k, v = torch.zeros((rows, H, D)), torch.randn((rows, H, D), generator=g)
    k[..., 0] = 2.0 ** 15
    k[..., 32] = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6])[torch.randint(0, 8, (rows, H), generator=g)]
    hpd.kv_append_fp4(pool, 0, k.to(DEV), v.to(DEV), torch.arange(rows, device=DEV))
    q = torch.zeros((B, 4, D), dtype=dtype, device=DEV)
    q[..., 0], q[..., 32] = 2.0 ** 15, 2.0 ** 8  # a code's half is a step of 2^30 in f32
    q[::3, :, 0] = 0
    ctx, tables, half = torch.tensor(lens, device=DEV), tables.to(DEV), torch.finfo(dtype).eps / 2
    for scale in (2.0 ** (power - 30), -2.0 ** (power - 30)):
        got = entry(q, pool, tables, ctx, 0, scale, torch.empty_like(q))
        out, A, _, most = reference(q, pool, tables, ctx, 0, scale)
        cut = 2.0 ** -26 if dtype == F32 else 2.0 ** -17
        tol = (16 * U + 2 * (most + 32) * U + cut) * A + half * out.abs() + 2.0 ** -25 * (dtype == F16)
        tol += most * 2.0 ** -118 * float(v.abs().amax())
        off = (got.double() - out).abs()
        assert not torch.isnan(got).any()
        assert (off <= tol).all(), f"worst {float((off / tol.clamp_min(1e-300)).max()):.3g} of the tolerance"


@DTYPES
@ROUTES
def test_values_near_the_largest_number(route, dtype):
    """Keys somewhat above the running maximum, later: a weight times its value must not
    overflow where the softmax's sum does not."""
    S, n, B = 16, 40, 3
    pool = gpu_pool(cpu_pool(1, B * n, S, 1, 64))
    k, v = torch.zeros((2, B * n * S, 1, 64))
    k[..., 0], v[:] = -24, 2.0 ** 127 if dtype != F16 else 6 * 2.0 ** 13
    v[..., ::2] *= -1
    for b, later in enumerate((40, 8 * 32 + 3, 600)):
        k[b * n * S, 0, 0], k[b * n * S + later, 0, 0] = 0, 4
    hpd.kv_append_fp4(pool, 0, k.to(DEV), v.to(DEV), torch.arange(B * n * S, device=DEV))
    tables, ctx = torch.arange(B * n, device=DEV).view(B, n), torch.full((B,), n * S - 3, device=DEV)
    q = torch.zeros((B, 2, 64), dtype=dtype, device=DEV)
    q[..., 0] = 8
    case = (q, pool, tables, ctx, 0)
    check(hpd.paged_attention_fp4_hip(*case), *case)


@ROUTES
@pytest.mark.parametrize("sign", [1, -1])
def test_f32_queries_up_to_the_largest_number(sign, route):
    """Such a query rounds up to no bf16 number; its terms must add up to it all the same."""
    S, n = 16, 5
    g = torch.Generator().manual_seed(5)
    pool = gpu_pool(cpu_pool(1, n, S, 1, 64))
    k, v = torch.zeros((n * S, 1, 64)), torch.randn((n * S, 1, 64), generator=g)
    k[..., 3] = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6])[torch.randint(0, 8, (n * S, 1), generator=g)] * 2.0 ** -100
    hpd.kv_append_fp4(pool, 0, k.to(DEV), v.to(DEV), torch.arange(n * S, device=DEV))
    tables, ctx = torch.arange(n, device=DEV)[None], torch.tensor([n * S - 2], device=DEV)
    q = torch.zeros((1, 2, 64), device=DEV)
    q[0, 0, 3], q[0, 1, 3] = sign * torch.finfo(F32).max, sign * 1.999 * 2.0 ** 126
    got = entry(q, pool, tables, ctx, 0, 2.0 ** -28, torch.empty_like(q))
    check(got, q, pool, tables, ctx, 0, 2.0 ** -28)


@DTYPES
@ROUTES
def test_tiny_queries_and_large_keys(route, dtype):
    """Queries whose further terms are no normal numbers. bf16's least number is 2^-133: of an f32
    query less than that is left out, and a score is off by up to 2^-133 max |k|, by which
    the weight and the sum that divides it are each off."""
    S, n, low = 16, 5, -20 if dtype == F16 else -122
    g = torch.Generator().manual_seed(6)
    pool = gpu_pool(cpu_pool(1, n, S, 1, 64))
    k, v = torch.zeros((n * S, 1, 64)), torch.randn((n * S, 1, 64), generator=g)
    k[..., 3] = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6])[torch.randint(0, 8, (n * S, 1), generator=g)] * 2.0 ** -low
    hpd.kv_append_fp4(pool, 0, k.to(DEV), v.to(DEV), torch.arange(n * S, device=DEV))
    tables, ctx = torch.arange(n, device=DEV)[None], torch.tensor([n * S - 2], device=DEV)
    q = torch.zeros((1, 4, 64), dtype=dtype, device=DEV)
    q[0, :, 3] = (torch.tensor([1.9999, 1.2345678, -1.7182818, 0.9876543]) * 2.0 ** low).to(dtype)
    got = entry(q, pool, tables, ctx, 0, 1.0, torch.empty_like(q))
    if dtype != F32:
        return check(got, q, pool, tables, ctx, 0, 1.0)
    out, A, X, n = reference(q, pool, tables, ctx, 0, 1.0)
    lost = 2.0 ** -133 * float(k.abs().amax())
    tol = (2 * 68 * U * X + 8 * U + 2 * (n + 32) * U + 2.0 ** -26 + 2 * lost) * A + U * out.abs()
    assert ((got.double() - out).abs() <= tol).all()


@ROUTES
@pytest.mark.parametrize("scale", [1e-45, -1e-38, 1e20, -1.7e38])
def test_scales_at_the_ends_of_the_range(scale, route):
    """Down to scales that make every weight equal, up to ones that leave the largest score alone."""
    q, pool, tables, ctx, layer = make(3, 4, 2, 64, 16, [300, 1, 77], F32, seed=15)
    scale = torch.tensor(scale, dtype=F32).item()
    if abs(scale) > 1:  # scores without an error: one dim of the keys
        q = torch.zeros_like(q)
        q[..., 5] = 1
    got = entry(q, pool, tables, ctx, layer, scale, torch.empty_like(q))
    out, A, _, n = reference(q, pool, tables, ctx, layer, scale)
    tol = (16 * U + 2 * (n + 32) * U + 2.0 ** -26) * A + U * out.abs()
    assert not torch.isnan(got).any()
    assert ((got.double() - out).abs() <= tol).all()
