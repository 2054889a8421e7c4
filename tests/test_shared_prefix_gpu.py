"""paged_attention_shared_prefix_hip against the softmax in 64 bits: the split form,
its shared tiles from registers and from LDS, and the one-launch form, grouped heads, rows shorter than the shared blocks, NaN
in every slot no row holds, masked entries, odd block sizes and strides, scores of
-inf, graphs and streams, and a rotary decode step through the pool.

Tolerance. With A = sum_t w_t |V_t| (w the softmax weights), u = 2^-24 and n keys:
 - a score is a chain of D fused terms: off by at most D u X, X = scale sum_d
   |q_d k_d|; scaling, the exponent's difference and exp2 add 4 u (1 + X); a weight
   and the sum that divides it are each off by that: 2 (D + 4) u max_t X + 8 u;
 - n fused additions into output and sum, joined over pieces: 2 (n + 32) u;
 - 2-byte types: every weight rounded, at most eps / 2 of it: eps / 2 of A;
 - the output's rounding: eps / 2 of itself (f32: u)."""
from __future__ import annotations

import math

import pytest
import torch

from minivllm import _ctypes_ops, _native
from minivllm import hip_paged_decode as hpd
from minivllm.kv_block_pool import KVBlockPool

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
ROUTES = pytest.mark.parametrize("route", ["registers", "lds", "one"])


@pytest.fixture(autouse=True)
def _route(request, monkeypatch):
    route = request.node.callspec.params.get("route") if hasattr(request.node, "callspec") else None
    if route:  # (f32, wide heads and block sizes that are no multiple of 16 keep to registers)
        monkeypatch.setenv("MINIVLLM_HIP_SHARED_SPLIT", "0" if route == "one" else "1")
        monkeypatch.setenv("MINIVLLM_HIP_SHARED_LDS", "1" if route == "lds" else "0")


def make(B, Hq, Hk, D, S, shared, ctx, dtype, seed=0, layers=2, layer=1, itype=torch.int64):
    """q, pool, tables, lengths over a permuted pool with NaN in every slot that no row holds."""
    g = torch.Generator().manual_seed(seed)
    M = max(1, shared, max(-(-max(0, c) // S) for c in ctx))
    need = [max(0, -(-c // S) - shared) for c in ctx]
    N = shared + sum(need) + 3
    perm = torch.randperm(N, generator=g)
    tables = torch.full((B, M), -1, dtype=torch.int64)
    tables[0, :shared] = perm[:shared]  # the other rows' shared entries stay -1: they are not read
    at = shared
    used = torch.zeros((N, S), dtype=torch.bool)
    longest = max(ctx)
    for i in range(shared):
        used[perm[i], :max(0, min(S, longest - i * S))] = True
    for b in range(B):
        for i in range(need[b]):
            tables[b, shared + i] = perm[at]
            used[perm[at], :max(0, min(S, ctx[b] - (shared + i) * S))] = True
            at += 1
    pool = KVBlockPool(layers, N, S, Hk, D, device=DEV, dtype=dtype)
    for t in (pool.k, pool.v):
        t.fill_(float("nan"))
        x = torch.randn((N, S, Hk, D), generator=g)
        x[~used] = float("nan")
        t[layer] = x.to(dtype).to(DEV)
    q = torch.randn((B, Hq, D), generator=g).to(dtype).to(DEV)
    return q, pool, tables.to(itype).to(DEV), torch.tensor(ctx, dtype=itype, device=DEV), layer


def reference(q, pool, tables, ctx, layer, shared, scale=None):
    """(out, A, X, n) in 64 bits; a row without keys gives 0."""
    B, Hq, D = q.shape
    _, N, S, Hk, _ = pool.k.shape
    G, M = Hq // Hk, tables.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros((B, Hq, D), dtype=torch.float64, device=DEV)
    A, X, most = torch.zeros_like(out), torch.zeros((B, Hq, 1), dtype=torch.float64, device=DEV), 0
    for b in range(B):
        c = min(max(int(ctx[b]), 0), M * S)
        t = torch.arange(c, device=DEV)
        blk = t // S
        row = torch.where(blk < shared, tables[0, blk], tables[b, blk]).long()
        ok = (row >= 0) & (row < N)
        row, off = row[ok], (t % S)[ok]
        if row.numel() == 0:
            continue
        most = max(most, row.numel())
        k = pool.k[layer, row, off].double().repeat_interleave(G, 1)  # [n, Hq, D]
        v = pool.v[layer, row, off].double().repeat_interleave(G, 1)
        s = (k * q[b].double()).sum(-1) * scale
        w = torch.softmax(s, 0)[..., None]
        out[b], A[b] = (w * v).sum(0), (w * v.abs()).sum(0)
        X[b, :, 0] = (k * q[b].double()).abs().sum(-1).amax(0) * abs(scale)
    return out, A, X, most


def check(got, want, dtype, what=""):
    out, A, X, n = want
    D = got.shape[-1]
    half = 0.5 * torch.finfo(dtype).eps
    bound = (2 * (D + 4) * U * X + 8 * U + 2 * (n + 32) * U) * A + half * out.abs()
    if dtype != F32:
        bound = bound + half * A
    bound = bound * 1.01 + torch.finfo(dtype).tiny * half
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} not finite"
    worst = ((got.double() - out).abs() / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


# (B, Hq, Hk, D, S, shared blocks, lengths): the shared tokens are shared * S.
CASES = {
    "one row one token": (1, 1, 1, 64, 16, 0, [1]),
    "one row shared only": (1, 4, 4, 64, 16, 1, [16]),
    "two short": (2, 2, 1, 128, 16, 2, [33, 40]),
    "lengths around the shared blocks": (9, 4, 4, 128, 16, 3, [48, 0, 1, 47, 49, 63, 64, 65, 200]),
    "all shorter than the shared blocks": (4, 6, 2, 64, 16, 4, [63, 5, 0, 40]),
    "no shared blocks": (5, 8, 2, 128, 16, 0, [1, 17, 300, 64, 0]),
    "grouped 8, tile ends inside": (7, 16, 2, 128, 16, 5, [81, 90, 100, 80, 333, 97, 112]),
    "many rows": (40, 6, 3, 64, 32, 9, [288 + 7 * i for i in range(40)]),
    "rows past one set": (70, 4, 2, 128, 16, 11, [176 + (i * 37) % 130 for i in range(70)]),
    "wide groups": (3, 40, 2, 64, 16, 6, [96, 130, 211]),
    "padded head dim": (6, 4, 2, 80, 16, 7, [112, 113, 150, 128, 90, 300]),
    "narrow heads": (4, 8, 8, 32, 16, 8, [200, 256, 131, 222]),
    "head dim 8": (3, 2, 2, 8, 16, 2, [40, 33, 32]),
    "wide heads": (5, 4, 2, 256, 16, 4, [64, 70, 100, 64, 150]),
    "wide padded heads": (20, 6, 3, 200, 32, 3, [96 + 9 * i for i in range(20)]),
    "block size 3": (4, 4, 2, 64, 3, 31, [93, 94, 120, 50]),
    "block size 1": (3, 2, 2, 128, 1, 70, [70, 71, 139]),
    "block size 24": (4, 6, 2, 128, 24, 3, [72, 80, 173, 96]),
    "block size 48": (4, 6, 6, 96, 48, 2, [96, 97, 250, 110]),
    "odd head dim": (4, 4, 2, 20, 16, 3, [48, 50, 64, 30]),
    "head dim 512": (3, 2, 1, 512, 16, 2, [32, 40, 33]),
    "long": (3, 4, 2, 128, 16, 130, [2080, 2500, 5000]),
    "hundreds of rows": (301, 2, 1, 64, 16, 3, [48 + (i * 31) % 140 if i % 9 else i % 50 for i in range(301)]),
    "teams of many sets": (150, 32, 2, 64, 16, 20, [320 + (i * 7) % 50 for i in range(150)]),
}


@DTYPES
@ROUTES
@pytest.mark.parametrize("name", CASES)
def test_against_64_bits(name, dtype, route):
    B, Hq, Hk, D, S, shared, ctx = CASES[name]
    q, pool, tables, lens, layer = make(B, Hq, Hk, D, S, shared, ctx, dtype, seed=len(name))
    got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=shared)
    again = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=shared)
    assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
    check(got, reference(q, pool, tables, lens, layer, shared), dtype, name)
    assert torch.equal(got, again)
    for b, c in enumerate(ctx):
        assert c > 0 or not got[b].any()


@DTYPES
@ROUTES
@pytest.mark.parametrize("B,H,shared,own", [(3, 1, 2_200_000, 5), (8, 8, 16, 41_000)], ids=["shared", "own"])
def test_windows_of_the_table_move_on(B, H, shared, own, dtype, route):
    """Runs of tiles past what one reading of the table covers (64 / 32 tiles a
    wavefront). Eight tokens, spread to the last, hold nearly all of the weight (their
    score is 25, 0 elsewhere), so a tile from a wrong place changes the output by about
    an eighth. An accumulator takes at most the keys of one of eight wavefronts: 2 (n / 8
    + 64) u of A and the rounding of weights and output."""
    D, S, P = 8, 16, -(-shared // 16)
    n = P * S + own
    g = torch.Generator(device=DEV).manual_seed(5)
    N = P + B * -(-own // S) + 2
    perm = torch.randperm(N, generator=g, device=DEV)
    tables = torch.empty((B, n // S + 1), dtype=torch.int32, device=DEV)
    tables[:, :P] = perm[:P]
    tables[:, P:] = perm[P:P + B * (tables.shape[1] - P)].view(B, -1)
    pool = KVBlockPool(1, N, S, H, D, device=DEV, dtype=dtype)
    pool.k.zero_()
    pool.v.normal_(generator=g)
    q = torch.zeros((B, H, D), dtype=dtype, device=DEV)
    q[..., 0] = 4
    at = torch.linspace(0, n - 1, 8, device=DEV, dtype=torch.float64).long()
    for b in range(B):
        pool.k[0, tables[b, at // S].long(), at % S, :, 0] = 25 * math.sqrt(D) / 4
    lens = torch.full((B,), n, device=DEV)
    got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, 0, shared_blocks=P)
    half, k = 0.5 * torch.finfo(dtype).eps, pool.k[0, :, :, 0, 0].double()
    for b in range(B):
        row = tables[b].long()
        w = torch.softmax((k[row] * 4 / math.sqrt(D)).flatten()[:n], 0)
        for h in range(H):
            v = pool.v[0, row, :, h].flatten(0, 1)[:n].double()
            out, A = (w[:, None] * v).sum(0), (w[:, None] * v.abs()).sum(0)
            bound = (2 * (n / 8 + 64) * U + 2 * (D + 4) * U * 26 + (half if dtype != F32 else 0)) * A + half * out.abs()
            assert ((got[b, h].double() - out).abs() <= 1.01 * bound).all(), (b, h)


@DTYPES
@ROUTES
def test_a_row_of_nan_keeps_to_itself(dtype, route):
    """NaN in one row's query, and in one row's own values, stays in that row; an
    infinite shared value is every row's, in its dim."""
    ctx = [100, 90, 130, 80, 64]
    q, pool, tables, lens, layer = make(5, 4, 2, 64, 16, 4, ctx, dtype, seed=12)
    want = reference(q, pool, tables, lens, layer, 4)
    q[1, 2, 5] = float("nan")
    pool.v[layer, tables[2, 7].long(), 3, 1, 9] = float("nan")
    pool.v[layer, tables[0, 2].long(), 6, 0, 30] = float("inf")
    got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=4)
    assert torch.isnan(got[1, 2]).all() and torch.isnan(got[2, 2:, 9]).all() and torch.isinf(got[[0, 2, 3, 4], :2, 30]).all()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[1, 2] = hit[2, 2:, 9] = hit[:, :2, 30] = True
    assert torch.isfinite(got[~hit]).all()
    out, A, X, n = want
    check(torch.where(hit, torch.zeros_like(got), got), (out.masked_fill(hit, 0), A, X, n), dtype)


def test_more_rows_than_the_split_takes():
    """4100 rows: one launch."""
    ctx = [20 + i % 30 for i in range(4100)]
    q, pool, tables, lens, layer = make(4100, 2, 1, 64, 16, 1, ctx, BF16, seed=13)
    assert _native.lib().mgi_paged_decode_shared_workspace_bytes(4100, 2, 1, 64, 16, tables.shape[1], 1, 1) == 0
    got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=1)
    pick = list(range(0, 4100, 37))
    row0 = tables[:1].expand(len(pick), -1)
    sub = torch.where(torch.arange(tables.shape[1], device=DEV) < 1, row0, tables[pick])
    check(got[pick], reference(q[pick], pool, sub, lens[pick], layer, 1), BF16)


@DTYPES
@ROUTES
def test_masked_entries_and_clamped_lengths(dtype, route):
    """Entries outside the pool mask their blocks, in the shared and in a row's own
    part; a row whose every entry is masked gives 0; lengths past the table and
    below 0 are clamped."""
    ctx = [160, 161, 320, 200, 175, 100]
    q, pool, tables, lens, layer = make(6, 6, 2, 128, 16, 10, ctx, dtype, seed=3, itype=torch.int32)
    N = pool.k.shape[1]
    tables[0, 3], tables[0, 9] = -1, N
    tables[2, 15], tables[3, 10] = N + 5, -7
    tables[2, 19] = -1
    lens[2], lens[5] = 100000, -4
    # The slots this row now reaches must be finite, where its blocks are.
    pool.k.nan_to_num_(0.25), pool.v.nan_to_num_(0.25)
    got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=10)
    check(got, reference(q, pool, tables, lens, layer, 10), dtype)
    assert not got[5].any()
    tables.fill_(-1)
    got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=10)
    assert not got.any()


@DTYPES
@ROUTES
def test_infinite_scores_and_values_in_unused_slots(dtype, route):
    """A score of -inf is a weight of 0, a row of nothing else NaN, as softmax has
    it; NaN or infinite keys and values past a length do not show (make() puts NaN
    there; infinities here)."""
    ctx = [64, 70, 33, 1, 96]
    q, pool, tables, lens, layer = make(5, 4, 4, 64, 16, 2, ctx, dtype, seed=9)
    pool.k.copy_(torch.where(pool.k.isnan(), torch.inf, pool.k)), pool.v.copy_(torch.where(pool.v.isnan(), -torch.inf, pool.v))
    q[..., 0] = q[..., 0].abs() + 0.5
    k = pool.k[layer]
    k[tables[0, 0].long(), 3, :, 0] = -torch.inf
    k[tables[1, 4].long(), 2, :, 0] = -torch.inf
    k[tables[4, 5].long(), :, :, 0] = -torch.inf
    k[tables[0, 0].long(), 0, :, 0] = -torch.inf  # all that row 3 holds
    got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=2)
    out, A, X, n = reference(q, pool, tables, lens, layer, 2)
    assert torch.isnan(got[3]).all() and torch.isnan(out[3]).all()
    rest = [0, 1, 2, 4]
    X = torch.full_like(X, 16.0)  # more than the finite keys have: 64 products of unit normals over 8
    check(got[rest], (out[rest], A[rest], X[rest], n), dtype)


@ROUTES
def test_large_scores(route):
    """Scores that differ by hundreds: late maxima rescale what came before."""
    ctx = [400, 321, 500]
    for dtype in (BF16, F32):
        q, pool, tables, lens, layer = make(3, 4, 2, 128, 16, 20, ctx, dtype, seed=4)
        ramp = torch.linspace(0.1, 30, 500, device=DEV)
        for b in range(3):
            for t in range(ctx[b]):
                e = tables[0 if t < 320 else b, t // 16].long()
                if t >= 320 or b == 0:
                    pool.k[layer, e, t % 16] *= ramp[t].to(dtype)
        got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=20)
        check(got, reference(q, pool, tables, lens, layer, 20), dtype, str(dtype))


@ROUTES
def test_strides_and_layouts(route):
    """q as a slice of a fused projection, transposed q, a pool whose heads come
    first or whose head dim is strided, tables and lengths strided: the same values."""
    ctx = [80, 90, 300, 64]
    q, pool, tables, lens, layer = make(4, 8, 2, 64, 16, 4, ctx, BF16, seed=5)
    want = reference(q, pool, tables, lens, layer, 4)
    wide = torch.full((4, 14, 64), float("nan"), dtype=BF16, device=DEV)
    wide[:, 3:11] = q
    wide_t = torch.stack((tables, tables * 0 - 1), -1)[..., 0]
    wide_l = torch.stack((lens, lens * 0), -1)[..., 0]
    heads_first = KVBlockPool(1, 1, 1, 1, 1, device=DEV, dtype=BF16)
    heads_first.k, heads_first.v = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (pool.k, pool.v))
    apart = KVBlockPool(1, 1, 1, 1, 1, device=DEV, dtype=BF16)
    apart.k, apart.v = (torch.stack((t, t), -1)[..., 1] for t in (pool.k, pool.v))
    call = lambda *x: hpd.paged_attention_shared_prefix_hip(*x, layer, shared_blocks=4)
    for name, args in {"slice": (wide[:, 3:11], pool, wide_t, wide_l),
                       "transposed": (q.transpose(0, 1).contiguous().transpose(0, 1), pool, tables, lens),
                       "dims apart": (q.transpose(1, 2).contiguous().transpose(1, 2), pool, tables, lens),
                       "heads first": (q, heads_first, tables, lens), "strided pool": (q, apart, tables, lens)}.items():
        check(call(*args), want, BF16, name)


@ROUTES
def test_any_finite_scale_through_the_c_entry(route):
    lib = _native.lib()
    ctx = [50, 49, 80, 20]
    for dtype in (F32, F16):
        q, pool, tables, lens, layer = make(4, 4, 2, 64, 16, 3, ctx, dtype, seed=6)
        L, N, S, H, D = pool.k.shape
        for scale in (0.3, -0.2, 0.0):
            out = torch.full_like(q, float("nan"))
            n = lib.mgi_paged_decode_shared_workspace_bytes(4, 4, 2, 64, S, tables.shape[1], 3, _native.DTYPE_CODES[dtype])
            ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device=DEV)
            _native.check(lib.mgi_paged_decode_shared(
                out.data_ptr(), _native.strides(out), q.data_ptr(), _native.strides(q), pool.k.data_ptr(), pool.v.data_ptr(),
                _native.strides(pool.k), _native.strides(pool.v), _native.DTYPE_CODES[dtype], tables.data_ptr(),
                _native.strides(tables), 1, lens.data_ptr(), 1, 1, 4, 4, 2, 64, S, N, tables.shape[1], L, layer, 3, scale,
                ws.data_ptr(), n, _native.stream_handle(DEV)))
            check(out, reference(q, pool, tables, lens, layer, 3, scale), dtype, f"{dtype} {scale}")


@ROUTES
def test_graph_replays_beside_eager_calls(route):
    """A captured call replayed on new inputs between eager ones: equal bits."""
    ctx = [100, 64, 150, 70, 99]
    q, pool, tables, lens, layer = make(5, 8, 4, 128, 16, 4, ctx, BF16, seed=7)
    pool.k.nan_to_num_(0.5), pool.v.nan_to_num_(0.5)
    call = lambda: hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).to(BF16).to(DEV))
        lens[2], lens[1] = 150 - 9 * i, 64 - 20 * i
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        check(out, reference(q, pool, tables, lens, layer, 4), BF16, f"replay {i}")


@ROUTES
def test_two_streams_at_once(route):
    ctx = [200 + 3 * i for i in range(30)]
    q, pool, tables, lens, layer = make(30, 8, 4, 128, 16, 10, ctx, F16, seed=8)
    call = lambda: hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=10)
    want = call()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_decode_steps_through_the_pool(interleaved):
    """A common prompt appended by kv_append_rope_hip, then decode steps of six
    sequences: rotary append and shared-prefix attention against the formulas in 64
    bits on the pool's own values, and against paged_attention_batch_hip."""
    B, H, D, S, P = 6, 4, 64, 16, 48
    table = hpd.rope_table(256, D, device=DEV)
    g = torch.Generator().manual_seed(21)
    rand = lambda *s: torch.randn(s, generator=g).to(BF16).to(DEV)
    pool = KVBlockPool(1, 40, S, H, D, device=DEV, dtype=BF16)
    pool.k.fill_(float("nan")), pool.v.fill_(float("nan"))
    perm = torch.randperm(40, generator=g)
    tables = torch.full((B, 6), -1)
    tables[:, :3] = perm[:3]
    tables[:, 3:] = perm[3:3 + 3 * B].view(B, 3)
    w = rand(D), rand(D)
    at = lambda b, t: int(tables[b, t // S]) * S + t % S
    x = rand(P, 3, H, D)
    hpd.kv_append_rope_hip(pool, 0, x[:, 0], x[:, 1], x[:, 2], torch.tensor([at(0, t) for t in range(P)], device=DEV),
                           torch.arange(P, device=DEV), table, *w, interleaved=interleaved)
    own = [0, 3, 15, 16, 1, 30]
    for step in range(35):
        length = [P + min(o, step) + 1 for o in own]
        pos = torch.tensor(length, device=DEV) - 1
        slots = torch.tensor([at(b, n - 1) for b, n in enumerate(length)], device=DEV)
        x = rand(B, 3, H, D)
        q = hpd.kv_append_rope_hip(pool, 0, x[:, 0], x[:, 1], x[:, 2], slots, pos, table, *w, interleaved=interleaved)
        lens, tab = pos + 1, tables.to(DEV)
        out = hpd.paged_attention_shared_prefix_hip(q, pool, tab, lens, 0, shared_blocks=3)
        if step % 7 == 0:
            check(out, reference(q, pool, tab, lens, 0, 3), BF16, f"step {step}")
            plain = hpd.paged_attention_batch_hip(q, pool, tab, lens, 0)
            assert (out.float() - plain.float()).abs().max() <= 2.0 ** -6 * (1 + plain.float().abs().max())


def test_ctypes_path_is_bit_identical_and_refuses_alike():
    ext = _native._load_extension()
    q, pool, tables, lens, layer = make(4, 8, 2, 64, 16, 4, [80, 64, 90, 10], BF16, seed=10)
    a, b = (o.paged_decode_shared(q, pool.k, pool.v, tables, lens, layer, 4) for o in (ext, _ctypes_ops))
    assert torch.equal(a, b)
    zero = KVBlockPool(1, 4, 0, 2, 64, device=DEV, dtype=BF16)
    grad = q.float().requires_grad_()
    bad = {"rank": (q[0], pool.k, pool.v, tables, lens, 1, 4), "heads": (q[:, :7], pool.k, pool.v, tables, lens, 1, 4),
           "dtype": (q.float(), pool.k, pool.v, tables, lens, 1, 4), "int": (q.int(), pool.k, pool.v, tables, lens, 1, 4),
           "head dim": (q[..., :32], pool.k, pool.v, tables, lens, 1, 4), "tables": (q, pool.k, pool.v, tables[:3], lens, 1, 4),
           "lengths": (q, pool.k, pool.v, tables, lens[:3], 1, 4), "table type": (q, pool.k, pool.v, tables.float(), lens, 1, 4),
           "length type": (q, pool.k, pool.v, tables, lens.float(), 1, 4), "layer": (q, pool.k, pool.v, tables, lens, 2, 4),
           "shared": (q, pool.k, pool.v, tables, lens, 1, 99), "negative": (q, pool.k, pool.v, tables, lens, 1, -1),
           "no columns": (q, pool.k, pool.v, tables[:, :0], lens, 1, 0), "empty": (q[:0], pool.k, pool.v, tables[:0], lens[:0], 1, 0),
           "block size": (q, zero.k, zero.v, tables, lens, 0, 0), "cpu": (q, pool.k, pool.v, tables.cpu(), lens, 1, 4),
           "pool": (q, pool.k, pool.v[:, :2], tables, lens, 1, 4),
           "gradient": (grad, pool.k.float(), pool.v.float(), tables, lens, 1, 4)}
    for name, args in bad.items():
        kind = RuntimeError if name == "gradient" else ValueError
        with pytest.raises(kind) as x:
            ext.paged_decode_shared(*args)
        with pytest.raises(kind) as y:
            _ctypes_ops.paged_decode_shared(*args)
        assert str(x.value) == str(y.value), name


@DTYPES
@ROUTES
@pytest.mark.parametrize("nats", [12.5, 17.5, 24.5])
def test_keys_far_below_a_sink_keep_their_weight(nats, dtype, route):
    """Every 32nd key scores ``nats`` above the others and has no value, so the output
    is the others', whose weights are 2^-18, 2^-25 and 2^-35 of the largest: below
    what f16 holds to half a step, unless scaled. Scaled by 2^13 they are off by
    half a step down to 2^-27 and by 2^-38 of the largest below, which adds 2^-38
    sum_t |V_t| / sum_t (w_t / max w)."""
    B, H, D, S, shared, ctx = 3, 2, 64, 16, 160, [3200, 2561, 3000]
    q, pool, tables, lens, layer = make(B, H, H, D, S, shared, ctx, dtype, seed=31)
    q.zero_()
    q[..., 0] = 4
    k, v = pool.k[layer], pool.v[layer]
    k.copy_(torch.where(k.isnan(), k, 0))
    v.mul_(100).add_(torch.where(v.isnan(), v, 1000))
    for b, c in enumerate(ctx):
        t = torch.arange(5, c, 32, device=DEV)
        row = torch.where(t // S < shared, tables[0, t // S], tables[b, t // S])
        k[row, t % S, :, 0], v[row, t % S] = 2 * nats, 0
    got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=shared)
    out, A, X, n = reference(q, pool, tables, lens, layer, shared)
    if dtype == F16:  # |V| < 1600, 31 of 32 keys; of the sum the sinks alone are n / 32
        A = A + 2.0 ** -38 * 1600 * 32 / (0.5 * torch.finfo(F16).eps)
    check(got, (out, A, X, n), dtype, f"{nats}")


@DTYPES
@ROUTES
@pytest.mark.parametrize("dims", [1, 6])
def test_scores_in_the_millions(dims, dtype, route):
    """Scores of 16 to 22 million, or 94 to 131 (2^27 is 134), thousands apart, exact
    in 32 bits: the largest key's value, to the rounding of its weight and of the output."""
    B, H, D, S, shared, ctx = 3, 2, 64, 16, 10, [300, 161, 259]
    q, pool, tables, lens, layer = make(B, H, H, D, S, shared, ctx, dtype, seed=32)
    q.zero_()
    q[..., :dims] = 61440
    g = torch.Generator().manual_seed(33)
    k, best = pool.k[layer], torch.empty((B, H, D), dtype=torch.float64, device=DEV)
    step = 32 if dtype == BF16 else 2  # of the type at 2048 .. 4096, doubled for bf16
    rank = torch.stack([torch.randperm(k.shape[0] * S, generator=g) for _ in range(H)], 1).view(-1, S, H).to(DEV)
    k.copy_(torch.where(k.isnan(), k, 0))
    k[..., :dims] = torch.where(k[..., :dims].isnan(), k[..., :dims], (2048 + step * (rank % (800 // step))).to(dtype)[..., None])
    for b, c in enumerate(ctx):
        t = torch.arange(c, device=DEV)
        row = torch.where(t // S < shared, tables[0, t // S], tables[b, t // S])
        for h in range(H):
            score, value = k[row, t % S, h, 0].double(), pool.v[layer, row, t % S, h].double()
            top = score == score.max()
            best[b, h] = value[top].mean(0)
            bound = value[top].abs().mean(0) * torch.finfo(dtype).eps * 1.01
            got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, layer, shared_blocks=shared)[b, h]
            assert ((got.double() - best[b, h]).abs() <= bound).all(), (b, h)


@DTYPES
@pytest.mark.parametrize("route", ["registers", "lds"])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_own_tiles_past_the_caches(D, dtype, route):
    """More than 192 MB of own keys and values (rows may name the same blocks): read
    as non-temporal, whole and padded head dims, runs that end inside tiles."""
    B, H, S, shared, N = 64, 16, 16, 3, 200
    g = torch.Generator().manual_seed(D)
    own = torch.randint(850, 1000, (B,), generator=g)
    own[7], own[20] = 0, -30  # no own tokens; shorter than the shared blocks
    assert (own.clamp_min(0) // 32 * 32).sum() * H * 2 * D * torch.finfo(dtype).bits // 8 > 192 << 20
    pool = KVBlockPool(1, N, S, H, D, device=DEV, dtype=dtype)
    pool.k.copy_(torch.randn(pool.k.shape, generator=g)), pool.v.copy_(torch.randn(pool.v.shape, generator=g))
    tables = torch.randint(0, N, (B, shared + 63), generator=g).to(DEV)
    lens = (own + shared * S).to(DEV)
    q = torch.randn((B, H, D), generator=g).to(dtype).to(DEV)
    got = hpd.paged_attention_shared_prefix_hip(q, pool, tables, lens, 0, shared_blocks=shared)
    check(got, reference(q, pool, tables, lens, 0, shared), dtype, f"{D}")
