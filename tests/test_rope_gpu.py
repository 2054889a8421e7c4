"""qk_norm_rope_hip and kv_append_rope_hip against the formula in 64 bits: the
chunked kernel (both chunk widths) and the one for any strides, head norms or
none, both pair orders, partial rotation, pool dtypes, skipped rows, graphs and
streams.

Tolerance. Everything is f32 up to one rounding to the output type, half a step
(eps / 2 of the value, or of the type's smallest normal below it). Before it: the
sum of squares is a chain of at most 16 fused terms and 6 additions (22 u, u =
2^-24, halved by the root), root, reciprocal, 1/D and eps 5 u, two products, and
the rotation's two products and a sum, each relative to the two terms' sizes: 11 +
5 + 2 + 2 = 20 u of |y_i| + |y_j|; 24 u allows for the cosine's use of a fused
product."""
from __future__ import annotations

import pytest
import torch

from minivllm import _ctypes_ops, _native
from minivllm import hip_paged_decode as hpd
from minivllm.kv_block_pool import KVBlockPool

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(dtype).to(DEV)


def _formula(x, w, rows, R, interleaved, eps):
    """(y, size): the result and the size of its terms, in 64 bits."""
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    i = torch.arange(R // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    c, s = rows[:, None, :R // 2].double(), rows[:, None, R // 2:].double()
    y, size = x.clone(), x.abs()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def _check(got, want, size, what):
    t = torch.finfo(got.dtype)
    bound = 24 * U * size + 0.5 * t.eps * want.abs().clamp_min(t.tiny) * 1.0001
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (err / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound"


def _bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


# (T, Hq, Hk, D, R): full and partial rotation, chunks of 8 and 4, dims without a chunk, one head, wide heads.
SHAPES = [(1, 8, 8, 32, 32), (5, 3, 1, 64, 32), (13, 16, 4, 128, 128), (3, 5, 5, 80, 80), (7, 4, 2, 80, 40),
          (300, 6, 2, 96, 96), (2, 2, 1, 256, 64), (2, 1, 1, 512, 512), (4, 3, 3, 20, 6), (3, 2, 2, 7, 2),
          (1030, 9, 1, 128, 64), (2, 130, 2, 128, 128)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,Hq,Hk,D,R", SHAPES)
def test_norm_rope_against_64_bits(dtype, T, Hq, Hk, D, R):
    table = hpd.rope_table(4000, R, device=DEV)
    qkv = _randn((T, Hq + 2 * Hk, D), dtype, 1, 3.0)
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hk]
    pos = torch.randint(0, 4000, (T,), generator=torch.Generator().manual_seed(2)).to(DEV)
    for wt in (None, dtype, F32):
        w = [None, None] if wt is None else [_randn((D,), wt, 3 + i) for i in range(2)]
        for inter in (False, True):
            qo, ko = hpd.qk_norm_rope_hip(q, k, pos, table, *w, eps=1e-5, interleaved=inter)
            for got, x, wi, n in ((qo, q, w[0], "q"), (ko, k, w[1], "k")):
                assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous()
                _check(got, *_formula(x, wi, table[pos], R, inter, 1e-5), f"{n} {wt} {inter}")


@pytest.mark.parametrize("D,R", [(128, 128), (64, 32)])
def test_any_strides_give_the_same_values(D, R):
    """Strided heads, head dims, rows and misaligned starts take the kernel for any
    strides, within the same bound; positions strided and int32."""
    T, Hq, Hk = 9, 4, 2
    table = hpd.rope_table(100, R + 6, device=DEV)[:, :R]  # rows further apart than they are long
    pos = torch.randint(0, 100, (T, 2), dtype=torch.int32, device=DEV)[:, 0]
    for dtype in (BF16, F32):
        base_q, base_k = _randn((T, Hq, D), dtype, 5), _randn((T, Hk, D), dtype, 6)
        w = _randn((D,), dtype, 7), _randn((D,), dtype, 8)
        views = {"dims apart": lambda x: x.transpose(0, 2).contiguous().transpose(0, 2),
                 "heads first": lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
                 "one element in": lambda x: torch.cat((x.new_zeros(1), x.flatten()))[1:].view(x.shape)}
        for name, view in views.items():
            q, k = view(base_q), view(base_k)
            qo, ko = hpd.qk_norm_rope_hip(q, k, pos, table, *w, interleaved=True)
            for got, x, wi in ((qo, q, w[0]), (ko, k, w[1])):
                _check(got, *_formula(x, wi, table[pos.long()], R, True, 1e-6), f"{name} {dtype}")
        row = base_q[:1].expand(T, Hq, D)  # one row for all positions
        qo, _ = hpd.qk_norm_rope_hip(row, base_k, pos, table)
        _check(qo, *_formula(row, None, table[pos.long()], R, False, 1e-6), "expanded row")


COMBOS = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16), (BF16, F32), (F16, F32)]


@pytest.mark.parametrize("new,pool_t", COMBOS, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("T,Hq,H,D,R,S", [(1, 8, 8, 32, 32, 16), (37, 8, 2, 128, 64, 16), (600, 4, 4, 64, 64, 3),
                                          (11, 3, 3, 20, 12, 4)])
def test_append_rope_writes_its_slots_and_nothing_else(new, pool_t, T, Hq, H, D, R, S):
    table = hpd.rope_table(9000, R, device=DEV)
    N, L, layer = -(-T // S) + 5, 3, 1
    pool = KVBlockPool(L, N, S, H, D, device=DEV, dtype=pool_t)
    pool.k.copy_(_randn(pool.k.shape, pool_t, 11))
    pool.v.copy_(_randn(pool.v.shape, pool_t, 12))
    before = pool.k.clone(), pool.v.clone()
    qkv = _randn((T, Hq + 2 * H, D), new, 13)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    g = torch.Generator().manual_seed(14)
    pos = torch.randint(0, 9000, (T,), generator=g)
    slots = torch.randperm(N * S, generator=g)[:T]
    if T > 10:
        slots[3], slots[7], pos[5], pos[6] = -1, N * S, 9000, -1
    off = (pos < 0) | (pos >= 9000)
    keep = (slots >= 0) & (slots < N * S) & ~off
    w = _randn((D,), new, 15), _randn((D,), new, 16)
    qo = hpd.kv_append_rope_hip(pool, layer, q, k, v, slots.to(DEV), pos.to(DEV), table, *w, interleaved=T == 37)
    rows = table[pos.clamp(0, 8999).to(DEV)]
    assert qo.dtype == pool_t
    want, size = _formula(q, w[0], rows, R, T == 37, 1e-6)
    _check(qo[~off.to(DEV)], want[~off.to(DEV)], size[~off.to(DEV)], "q")
    assert torch.isnan(qo[off.to(DEV), :, :R]).all()
    if R < D and off.any():
        _check(qo[off.to(DEV), :, R:], want[off.to(DEV), :, R:], size[off.to(DEV), :, R:], "q past R")
    flat = lambda t: t[layer].view(N * S, H, D)
    at, kept = slots[keep].to(DEV), keep.to(DEV)
    want, size = _formula(k, w[1], rows, R, T == 37, 1e-6)
    _check(flat(pool.k)[at], want[kept], size[kept], "k")
    assert torch.equal(_bits(flat(pool.v)[at]), _bits(v[kept].to(pool_t)))
    for new_t, old in zip((pool.k, pool.v), before):
        flat(old)[at] = flat(new_t)[at]
        assert torch.equal(_bits(new_t), _bits(old))


def test_append_rope_odd_pools_and_repeated_slots():
    """A pool whose head dim is strided (a view), and two rows on one slot: each of
    K and V is one row's, whole."""
    T, H, D = 6, 2, 64
    pool = KVBlockPool(1, 4, 4, H, D, device=DEV, dtype=BF16)
    wide = torch.zeros((1, 4, 4, H, D, 2), dtype=BF16, device=DEV)
    pool.k, pool.v = wide[..., 0], wide[..., 1]
    table = hpd.rope_table(64, D, device=DEV)
    q, k, v = (_randn((T, H, D), BF16, 20 + i) for i in range(3))
    pos = torch.arange(T, device=DEV)
    slots = torch.tensor([0, 5, 9, 9, 15, 2], device=DEV)
    hpd.kv_append_rope_hip(pool, 0, q, k, v, slots, pos, table)
    want, size = _formula(k, None, table[pos], D, False, 0.0)
    kk, vv = pool.k[0].reshape(16, H, D), pool.v[0].reshape(16, H, D)
    for i in (0, 1, 4, 5):
        _check(kk[slots[i]][None], want[i][None], size[i][None], f"row {i}")
        assert torch.equal(vv[slots[i]], v[i])
    assert any(torch.equal(vv[9], v[i]) for i in (2, 3))
    both = [(kk[9].double() - want[i]).abs().max() < 0.05 for i in (2, 3)]
    assert any(both)
    rest = [s for s in range(16) if s not in slots.tolist()]
    assert not kk[rest].any() and not vv[rest].any()


def test_infinities_past_the_rotated_dims_and_nan_values():
    """Dims past R are the input's own; a NaN or infinity stays in its own head."""
    T, H, D, R = 4, 3, 128, 64
    q = _randn((T, H, D), F16, 30)
    q[1, 2, 100], q[2, 0, 3], q[3, 1, 127] = float("inf"), float("nan"), float("-inf")
    table = hpd.rope_table(16, R, device=DEV)
    pos = torch.arange(T, device=DEV)
    qo, _ = hpd.qk_norm_rope_hip(q, q, pos, table)
    assert torch.equal(_bits(qo[..., R:]), _bits(q[..., R:]))
    hit = torch.zeros_like(qo, dtype=torch.bool)
    hit[2, 0, 3] = hit[2, 0, 35] = True
    assert torch.equal(torch.isnan(qo), hit)


def test_empty_calls_and_far_positions():
    table = hpd.rope_table(140000, 64, device=DEV)
    q = torch.empty((0, 4, 64), dtype=BF16, device=DEV)
    pos = torch.empty(0, dtype=torch.long, device=DEV)
    qo, ko = hpd.qk_norm_rope_hip(q, q[:, :2], pos, table)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)
    pool = KVBlockPool(1, 2, 4, 4, 64, device=DEV, dtype=BF16)
    assert hpd.kv_append_rope_hip(pool, 0, q, q, q, pos, pos, table).shape == (0, 4, 64)
    q = _randn((3, 4, 64), F32, 40)
    pos = torch.tensor([131071, 139999, 65536], device=DEV)
    qo, _ = hpd.qk_norm_rope_hip(q, q, pos, table)
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=DEV) / 32)
    angle = pos[:, None].double() * freq
    rows = torch.cat((angle.cos(), angle.sin()), 1)
    want, size = _formula(q, None, rows, 64, False, 0.0)
    _check(qo, want, size, "far")  # the table's own rounding is one more u of each term


def test_index_types_wide_strides_and_converted_nan_values():
    """int32 and strided positions and slots, and a stride past 31 bits (of a single
    row), give the bits of plain int64 ones; a NaN value converts as kv_append does."""
    T, Hq, H, D = 9, 4, 2, 128
    table = hpd.rope_table(64, D, device=DEV)
    q, k, v = _randn((T, Hq, D), F32, 90), _randn((T, H, D), F32, 91), _randn((T, H, D), F32, 92)
    v[3, 1, 5], v[4, 0, 0] = float("nan"), -float("nan")
    w = _randn((D,), F32, 93), _randn((D,), F32, 94)
    pos, slots = torch.arange(T, device=DEV) * 7, torch.tensor([3, 40, -1, 8, 30, 2, 99, 17, 0], device=DEV)
    pools = [KVBlockPool(1, 3, 16, H, D, device=DEV, dtype=BF16) for _ in range(4)]
    for p in pools:
        p.k.zero_(), p.v.zero_()
    wide = lambda t: torch.stack((t, t + 1), 1)[:, 0]
    got = [hpd.kv_append_rope_hip(p, 0, q, k, v, s, i, table, *w)
           for p, s, i in zip(pools, (slots, slots.int(), wide(slots)), (pos, wide(pos.int()), wide(pos)))]
    hpd.kv_append(pools[3], 0, k, v, slots)
    for p, out in zip(pools[1:3], got[1:]):
        assert torch.equal(_bits(out), _bits(got[0]))
        assert torch.equal(_bits(p.k), _bits(pools[0].k)) and torch.equal(_bits(p.v), _bits(pools[0].v))
    assert torch.equal(_bits(pools[3].v), _bits(pools[0].v))
    one = [t[:1].contiguous() for t in (q, k)]
    far = [t.as_strided(t.shape, (2 ** 31, D, 1)) for t in one]
    a, b = (hpd.qk_norm_rope_hip(*x, pos[1:2], table, *w) for x in (one, far))
    for x, y, src, wt in zip(a, b, one, w):
        want, size = _formula(src, wt, table[pos[1:2]], D, False, 1e-6)
        _check(x, want, size, "row")
        _check(y, want, size, "far row")


def test_graph_replays_and_streams():
    """Captured together, replayed on new inputs, equal to the eager calls; another
    stream than the tensors' own."""
    T, Hq, H, D = 24, 8, 2, 128
    table = hpd.rope_table(512, D, device=DEV)
    pool, twin = (KVBlockPool(1, 8, 16, H, D, device=DEV, dtype=BF16) for _ in range(2))
    for p in (pool, twin):
        p.k.zero_(), p.v.zero_()
    q, k, v = _randn((T, Hq, D), BF16, 50), _randn((T, H, D), BF16, 51), _randn((T, H, D), BF16, 52)
    w = _randn((D,), BF16, 53), _randn((D,), BF16, 54)
    slots, pos = torch.arange(T, device=DEV) * 3, torch.arange(T, device=DEV)
    call = lambda p: hpd.kv_append_rope_hip(p, 0, q, k, v, slots, pos, table, *w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(pool)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(pool)
        qn, kn = hpd.qk_norm_rope_hip(q, k, pos, table, *w)
    for i in range(4):
        q.copy_(_randn(q.shape, BF16, 60 + i))
        k.copy_(_randn(k.shape, BF16, 70 + i))
        pos.add_(5)
        graph.replay()
        eager = call(twin)
        torch.cuda.synchronize()
        assert torch.equal(_bits(out), _bits(eager)) and torch.equal(_bits(qn), _bits(eager))
        assert torch.equal(_bits(pool.k), _bits(twin.k)) and torch.equal(_bits(pool.v), _bits(twin.v))
        assert torch.equal(_bits(kn), _bits(pool.k[0].view(-1, H, D)[slots]))


def test_ctypes_path_is_bit_identical_and_refuses_alike():
    ext = _native._load_extension()
    table = hpd.rope_table(64, 64, device=DEV)
    q, k, v = _randn((5, 6, 64), BF16, 80), _randn((5, 2, 64), BF16, 81), _randn((5, 2, 64), BF16, 82)
    w = _randn((64,), F32, 83), _randn((64,), F32, 84)
    pos, slots = torch.arange(5, device=DEV), torch.tensor([0, 3, -1, 7, 9], device=DEV)
    pools = [KVBlockPool(1, 3, 4, 2, 64, device=DEV, dtype=F32) for _ in range(2)]
    for p in pools:
        p.k.zero_(), p.v.zero_()
    got = []
    for ops, p in zip((ext, _ctypes_ops), pools):
        got.append((*ops.qk_norm_rope(q, k, pos, table, *w, 1e-6, True),
                    ops.kv_append_rope(p.k, p.v, 0, q, k, v, slots, pos, table, *w, 1e-6, False), p.k, p.v))
    for a, b in zip(*got):
        assert torch.equal(_bits(a), _bits(b))
    p = pools[0]
    neg = torch.view_as_complex(_randn((5, 6, 64, 2), F32, 85)).conj().imag
    grad = q.float().requires_grad_()
    norm = [("rank", (q[0], k, pos, table, None, None, 1e-6, False)), ("rows", (q, k[:3], pos, table, None, None, 1e-6, False)),
            ("dtype", (q, k.float(), pos, table, None, None, 1e-6, False)), ("int q", (q.int(), k.int(), pos, table, None, None, 1e-6, False)),
            ("positions", (q, k, pos[:4], table, None, None, 1e-6, False)), ("float positions", (q, k, pos.float(), table, None, None, 1e-6, False)),
            ("table dtype", (q, k, pos, table.half(), None, None, 1e-6, False)), ("table stride", (q, k, pos, table.t().contiguous().t(), None, None, 1e-6, False)),
            ("odd R", (q, k, pos, table[:, :63], None, None, 1e-6, False)), ("wide R", (q[..., :32], k[..., :32], pos, table, None, None, 1e-6, False)),
            ("no rows", (q, k, pos, table[:0], None, None, 1e-6, False)), ("one weight", (q, k, pos, table, w[0], None, 1e-6, False)),
            ("weight shape", (q, k, pos, table, w[0][:32], w[1], 1e-6, False)), ("weight dtype", (q, k, pos, table, w[0].half(), w[1].half(), 1e-6, False)),
            ("weights differ", (q, k, pos, table, w[0], w[1].bfloat16(), 1e-6, False)), ("eps", (q, k, pos, table, *w, float("nan"), False)),
            ("eps sign", (q, k, pos, table, *w, -1e-6, False)), ("cpu positions", (q, k, pos.cpu(), table, *w, 1e-6, False)),
            ("no heads", (q[:, :0], k, pos, table, *w, 1e-6, False)), ("negated", (neg, neg, pos, table, None, None, 1e-6, False)),
            ("gradient", (grad, grad, pos, table, None, None, 1e-6, False))]
    app = [("heads", (p.k, p.v, 0, q, q, q, slots, pos, table, None, None, 1e-6, False)),
           ("v", (p.k, p.v, 0, q, k, v[:3], slots, pos, table, None, None, 1e-6, False)),
           ("v dtype", (p.k, p.v, 0, q, k, v.float(), slots, pos, table, None, None, 1e-6, False)),
           ("slots", (p.k, p.v, 0, q, k, v, slots[:2], pos, table, None, None, 1e-6, False)),
           ("slot dtype", (p.k, p.v, 0, q, k, v, slots.float(), pos, table, None, None, 1e-6, False)),
           ("layer", (p.k, p.v, 1, q, k, v, slots, pos, table, None, None, 1e-6, False)),
           ("pool", (p.k, p.v[:, :2], 0, q, k, v, slots, pos, table, None, None, 1e-6, False)),
           ("f16 to bf16", (p.k.bfloat16(), p.v.bfloat16(), 0, q.half(), k.half(), v.half(), slots, pos, table, None, None, 1e-6, False)),
           ("rank", (p.k, p.v, 0, q[0], k, v, slots, pos, table, None, None, 1e-6, False))]
    before = p.k.clone()
    for fn, calls in (("qk_norm_rope", norm), ("kv_append_rope", app)):
        for name, args in calls:
            kind = RuntimeError if name == "gradient" else ValueError
            with pytest.raises(kind) as a:
                getattr(ext, fn)(*args)
            with pytest.raises(kind) as b:
                getattr(_ctypes_ops, fn)(*args)
            assert str(a.value) == str(b.value), name
    assert torch.equal(p.k, before)


def _rows_on_few_slots(T, Hq, H, D, R, S, new, pool_t, strided, itype):
    """An append of T rows to few slots, some of them skipped: (per slot the rows
    that are written, in order; what the pool holds after; the rows' keys and their
    terms in 64 bits; the values as the pool's type)."""
    g = torch.Generator().manual_seed(T)
    N, P = max(2, -(-T // (3 * S))), 500
    table = hpd.rope_table(P, R, device=DEV)
    pool = KVBlockPool(2, N, S, H, D, device=DEV, dtype=pool_t)
    if strided:
        pool.k, pool.v = (torch.zeros((2, N, S, H, D, 2), dtype=pool_t, device=DEV)[..., 1] for _ in range(2))
    pool.k.fill_(7), pool.v.fill_(7)
    q, k, v = (_randn((T, h, D), new, 100 + i) for i, h in enumerate((Hq, H, H)))
    w = _randn((D,), new, 103), _randn((D,), new, 104)
    pos, few = torch.randint(0, P, (T,), generator=g), torch.randperm(N * S, generator=g)[:max(1, T // 4)]
    slots = few[torch.randint(0, few.numel(), (T,), generator=g)]
    slots[torch.rand(T, generator=g) < 0.05] = -1
    if itype == torch.int64:  # past the pool, the low word a slot's
        slots[torch.rand(T, generator=g) < 0.1] += 2 ** 32
    pos[torch.rand(T, generator=g) < 0.2] = P  # not written: the row before on its slot stays
    hpd.kv_append_rope_hip(pool, 1, q, k, v, slots.to(itype).to(DEV), pos.to(itype).to(DEV), table, *w)
    rows = [[t for t in range(T) if slots[t] == s and pos[t] < P] for s in range(N * S)]
    assert T < 13 or any(len(r) > 1 for r in rows)
    want, size = _formula(k, w[1], table[pos.clamp_max(P - 1).to(DEV)], R, False, 1e-6)
    flat = [t[1].reshape(N * S, H, D) for t in (pool.k, pool.v)]
    assert (pool.k[0] == 7).all() and (pool.v[0] == 7).all()
    for s, r in enumerate(rows):
        if not r:
            assert (flat[0][s] == 7).all() and (flat[1][s] == 7).all()
    return rows, *flat, want, size, v.to(pool_t)


@pytest.mark.parametrize("itype", [torch.int64, torch.int32], ids=["i64", "i32"])
@pytest.mark.parametrize("T", [2, 13, 64, 65, 200, 256])
@pytest.mark.parametrize("Hq,H,D,R,S,new,pool_t,strided", [
    (8, 4, 128, 128, 16, BF16, BF16, False), (2, 1, 64, 24, 4, F32, F16, False), (1, 1, 16, 16, 3, F16, F16, False),
    (3, 2, 20, 6, 4, BF16, F32, False), (2, 2, 64, 64, 4, BF16, BF16, True)])
def test_of_rows_on_one_slot_the_last_written_is_kept(T, itype, Hq, H, D, R, S, new, pool_t, strided):
    rows, kk, vv, want, size, v = _rows_on_few_slots(T, Hq, H, D, R, S, new, pool_t, strided, itype)
    at = [s for s, r in enumerate(rows) if r]
    last = [rows[s][-1] for s in at]
    _check(kk[at], want[last], size[last], "k")
    assert torch.equal(_bits(vv[at]), _bits(v[last]))


@pytest.mark.parametrize("strided", [False, True])
def test_longer_calls_keep_one_of_the_rows_in_every_element(strided):
    rows, kk, vv, want, size, v = _rows_on_few_slots(400, 4, 2, 64, 64, 16, BF16, BF16, strided, torch.int64)
    for s, r in enumerate(rows):
        if r:
            bound = 24 * U * size[r] + 2.0 ** -8 * want[r].abs().clamp_min(torch.finfo(BF16).tiny) * 1.0001
            assert ((kk[s].double() - want[r]).abs() <= bound).any(0).all(), s
            assert (vv[s] == v[r]).any(0).all(), s
