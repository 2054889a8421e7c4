"""prompt_attention_hip against the softmax in 64 bits: grouped heads, lengths around the
tiles, empty sequences, rows of no sequence, what is not a number in places that a row
does not see, strides, graphs and streams, and a request's life with a 4-bit cache.

Tolerance. With A = sum_j w_j |v_j| (w the softmax weights), u = 2^-24 and n keys:
 - a score is a sum of D products in f32: off by at most D u X, X = scale sum_d
   |q_d k_d|; scaling, the exponent's difference and exp2 add 4 u (1 + X); a weight and
   the sum that divides it are each off by that: 2 (D + 4) u max_j X + 8 u;
 - n additions into output and sum: 2 (n + 32) u;
 - 2-byte types: every weight rounded to its type, at most eps / 2 of it, in the output
   and in the sum that divides: 2 (eps / 2) of A (f16 weights are scaled so that those of
   2^-27 and more are normal numbers: at most 2^-38 each below that, n 2^-38 max |v|);
 - the output's rounding: eps / 2 of itself (f32: u), in f16 2^-25 where it is subnormal."""
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


def make(lens, Hq, Hk, D, dtype, seed=0, lead=0, tail=0, itype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    T = lead + sum(lens) + tail
    qkv = torch.randn((T, Hq + 2 * Hk, D), generator=g).to(dtype).to(DEV)
    cu = torch.tensor([lead] + lens).cumsum(0).to(itype).to(DEV)
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], cu


def reference(q, k, v, cu, scale=None):
    """(out, A, X) in 64 bits; rows of no sequence are 0."""
    T, Hq, D = q.shape
    Hk = k.shape[1]
    G = Hq // Hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros((T, Hq, D), dtype=torch.float64, device=DEV)
    A, X = torch.zeros_like(out), torch.zeros((T, Hq, 1), dtype=torch.float64, device=DEV)
    ends = cu.tolist()
    for lo, hi in zip(ends, ends[1:]):
        n = hi - lo
        if n <= 0:
            continue
        hidden = torch.ones((n, n), dtype=torch.bool, device=DEV).triu(1)
        for h in range(Hq):
            qh, kh, vh = q[lo:hi, h].double() * scale, k[lo:hi, h // G].double(), v[lo:hi, h // G].double()
            w = torch.softmax((qh @ kh.t().contiguous()).masked_fill(hidden, -math.inf), 1)
            out[lo:hi, h], A[lo:hi, h] = w @ vh, w @ vh.abs()
            X[lo:hi, h] = (qh.abs() @ kh.abs().t().contiguous()).masked_fill(hidden, 0).amax(1, keepdim=True)
    return out, A, X


def tolerance(q, v, cu, out, A, X):
    D, half = q.shape[2], torch.finfo(q.dtype).eps / 2
    n = int((cu[1:] - cu[:-1]).max()) if len(cu) > 1 else 0
    tol = (2 * (D + 4) * U * X + 8 * U + 2 * (n + 32) * U) * A + half * out.abs()
    if q.dtype != F32:
        tol = tol + 2 * half * A
    if q.dtype == F16:
        tol = tol + n * 2.0 ** -38 * float(v.abs().amax()) + 2.0 ** -25
    return tol


def check(got, q, k, v, cu, scale=None):
    out, A, X = reference(q, k, v, cu, scale)
    off, tol = (got.double() - out).abs(), tolerance(q, v, cu, out, A, X)
    assert got.shape == q.shape and got.dtype == q.dtype and not torch.isnan(got).any()
    assert (off <= tol).all(), f"worst {float((off / tol.clamp_min(1e-300)).max()):.3g} of the tolerance"


LENS = [1, 0, 31, 32, 33, 130, 64, 65, 200]


@DTYPES
@pytest.mark.parametrize("Hq,Hk,D", [(1, 1, 128), (8, 2, 128), (6, 3, 64), (3, 3, 32), (4, 1, 80), (12, 1, 96), (2, 1, 256),
                                     (5, 1, 192), (2, 2, 8), (4, 4, 136), (8, 1, 48), (2, 1, 20), (3, 1, 1), (4, 2, 253),
                                     (2, 1, 125), (4, 1, 70), (2, 2, 90), (1, 1, 190)])
def test_lengths_heads_dims(Hq, Hk, D, dtype):
    case = make(LENS, Hq, Hk, D, dtype, seed=Hq + D)
    check(hpd.prompt_attention_hip(*case), *case)


@DTYPES
def test_long_prompts(dtype):
    case = make([1500, 5, 700], 4, 1, 128, dtype, seed=1)
    check(hpd.prompt_attention_hip(*case), *case)
    case = make([1111], 2, 2, 64, dtype, seed=2)
    check(hpd.prompt_attention_hip(*case), *case)


def test_many_sequences():
    lens = [(i * 7) % 45 for i in range(300)]
    lens[201] = 600
    case = make(lens, 4, 2, 64, BF16, seed=3, itype=torch.int32)
    check(hpd.prompt_attention_hip(*case), *case)


@DTYPES
def test_rows_of_no_sequence_are_zero(dtype):
    q, k, v, cu = make([40, 0, 70], 4, 2, 64, dtype, lead=9, tail=100)
    got = hpd.prompt_attention_hip(q, k, v, cu)
    check(got, q, k, v, cu)
    assert (got[:9] == 0).all() and (got[119:] == 0).all()
    for empty in ([], [0, 0, 0]):
        cu = torch.tensor([0] + empty, device=DEV)
        assert (hpd.prompt_attention_hip(q, k, v, cu) == 0).all()


def entry(q, k, v, cu, out, scale, zero_rest):
    T, Hq, D = q.shape
    _native.check(_native.lib().mgi_prompt_attention(
        out.data_ptr(), _native.strides(out), q.data_ptr(), _native.strides(q), k.data_ptr(), _native.strides(k),
        v.data_ptr(), _native.strides(v), _native.DTYPE_CODES[q.dtype], cu.data_ptr(), cu.stride(0),
        _native.ITYPE_CODES[cu.dtype], len(cu) - 1, T, Hq, k.shape[1], D, scale, zero_rest, _native.stream_handle(DEV)))
    return out


@DTYPES
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 0.5])
def test_any_scale_and_strides(scale, dtype):
    q, k, v, cu = make([50, 77, 3], 4, 2, 40, dtype, lead=5, tail=6)
    q, k = q.transpose(0, 2).contiguous().transpose(0, 2), k.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((len(q) + 1, 6, 90), 7.0, dtype=dtype, device=DEV)
    out = wide[:-1, 1:5, 3:83:2]
    entry(q, k, v, cu[None].repeat(2, 1).t().contiguous()[:, 1], out, scale, 0)
    assert (out[:5] == 7).all() and (out[-6:] == 7).all()  # left as they were
    body = torch.zeros_like(out)
    body[5:-6] = out[5:-6]
    check(body, q, k, v, cu, scale)
    out.fill_(7.0)
    assert (wide == 7).all()  # nothing beside the rows


def test_starts_outside_the_rows_are_clamped():
    q, k, v, _ = make([100], 2, 1, 64, F32)
    cu = torch.tensor([-50, 30, 90, 1 << 40], device=DEV)
    check(hpd.prompt_attention_hip(q, k, v, cu), q, k, v, cu.clamp(0, 100))
    hpd.prompt_attention_hip(q, k, v, torch.tensor([0, 90, 20, 100, 5], device=DEV))  # falling: in bounds, no more


@DTYPES
@pytest.mark.parametrize("Hq,Hk", [(4, 1), (2, 1), (1, 1)])
def test_what_a_row_does_not_see_does_not_matter(Hq, Hk, dtype):
    lens = [70, 150, 33]
    q, k, v, cu = make(lens, Hq, Hk, 64, dtype, seed=8)
    clean = hpd.prompt_attention_hip(q, k, v, cu)
    k, v = k.clone(), v.clone()
    k[69], v[69], v[70 + 140], v[70 + 149, 0, 5] = float("nan"), float("inf"), float("nan"), -float("inf")
    v[220 + 3, 0, 7], k[220 + 32] = float("inf"), float("nan")
    got = hpd.prompt_attention_hip(q, k, v, cu)
    # An output that did not see it is what it was, up to another order of the same sums.
    out, A, X = reference(q, torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0), cu)
    tol = tolerance(q, torch.nan_to_num(v, 0, 0, 0), cu, out, A, X)
    off = (got.double() - clean.double()).abs()
    rows = torch.ones(sum(lens), dtype=torch.bool, device=DEV)
    rows[69], rows[70 + 140:220], rows[220 + 3:] = False, False, False
    assert (off[rows] <= 2 * tol[rows]).all()
    assert torch.isnan(got[69]).all() and torch.isnan(got[70 + 140:220]).all() and torch.isnan(got[220 + 32]).all()
    # One infinite element of one value: that dim of every row from there on.
    mid = slice(220 + 3, 220 + 32)
    keep = torch.arange(64, device=DEV) != 7
    assert (got[mid, :, 7] == float("inf")).all()
    assert (off[mid][..., keep] <= 2 * tol[mid][..., keep]).all()


@DTYPES
def test_large_scores(dtype):
    q, k, v, cu = make([300, 90], 4, 2, 64, dtype, seed=9)
    check(hpd.prompt_attention_hip(q * 40, k, v, cu), q * 40, k, v, cu)


@DTYPES
def test_weights_far_below_the_largest_keep_their_share(dtype):
    """One key far above thousands that hold half of the mass together."""
    n, D = 4096, 64
    q, k, v = (torch.zeros((n, 1, D), dtype=dtype, device=DEV) for _ in range(3))
    q[:, 0, 0] = 1
    k[0, 0, 0] = 8 * 12 * math.log(2)  # score 12 ln 2: a weight of 2^12 beside those of 1
    v[1:, 0, 1] = 1
    cu = torch.tensor([0, n], device=DEV)
    check(hpd.prompt_attention_hip(q, k, v, cu), q, k, v, cu)


def test_same_inputs_same_bits_and_ctypes():
    case = make([500, 1, 0, 90, 1200, 33], 8, 2, 128, BF16)
    first = hpd.prompt_attention_hip(*case)
    for _ in range(5):
        assert torch.equal(first, hpd.prompt_attention_hip(*case))
    assert torch.equal(first, _ctypes_ops.prompt_attention(*case))


def test_offsets_past_32_bits():
    """Rows 2^31 elements and more apart."""
    T, wide = 40, 60_000_000
    base = torch.empty(T * wide, dtype=BF16, device=DEV)
    q, k, v, cu = make([T], 2, 1, 64, BF16)
    far = [torch.as_strided(base, x.shape, (wide, 64, 1), i * 1024) for i, x in enumerate((q, k, v))]
    for x, y in zip(far, (q, k, v)):
        x.copy_(y)
    check(hpd.prompt_attention_hip(*far, cu), *far, cu)


def test_graph_replays_follow_the_starts():
    q, k, v, cu = make([300, 40, 172], 8, 2, 128, BF16)
    q, k, v = q.clone(), k.clone(), v.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        hpd.prompt_attention_hip(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hpd.prompt_attention_hip(q, k, v, cu)
    for starts in ([0, 300, 340, 512], [0, 1, 500, 512], [0, 0, 512, 512], [7, 50, 60, 100]):
        cu.copy_(torch.tensor(starts, device=DEV))
        q.normal_()
        graph.replay()
        got = out.clone()
        want = hpd.prompt_attention_hip(q, k, v, cu)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        check(got, q, k, v, cu)


def test_calls_on_two_streams_at_once():
    cases = [make([900, 30, 411], 8, 2, 128, BF16, seed=s) for s in (1, 2)]
    want = [hpd.prompt_attention_hip(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(hpd.prompt_attention_hip(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    q, k, v, cu = make([20, 30], 4, 2, 64, BF16)
    for f in (_native.ops().prompt_attention, _ctypes_ops.prompt_attention):
        for args, msg in [((q[0], k, v, cu), "shape"), ((q.double(), k, v, cu), "float32"), ((q, k.float(), v, cu), "share"),
                          ((q, k, v[:, :1], cu), "matching"), ((q[:, :3], k, v, cu), "divide"), ((q[1:], k, v, cu), "rows"),
                          ((q, k, v, cu[:0]), r"\[B\+1\]"), ((q, k, v, cu.float()), "integer"), ((q, k, v, cu.cpu()), "same GPU"),
                          ((q[..., :0], k[..., :0], v[..., :0], cu), "nonzero"), ((q[..., :32], k, v, cu), "head dimension")]:
            with pytest.raises(ValueError, match=msg):
                f(*args)
        wide = torch.zeros((2, 1, 264), dtype=BF16, device=DEV)
        with pytest.raises(ValueError, match="256"):
            f(wide, wide, wide, cu)
        with pytest.raises(RuntimeError, match="inference-only"):
            f(q.clone().requires_grad_(), k, v, cu)
        assert f(q[:0], k[:0], v[:0], cu).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_a_requests_life_with_a_4_bit_cache(dtype):
    """Prompts attend over their own keys and values and go into the 4-bit pool; decode
    steps append and attend there. Against the same in 64 bits over the values that the pool
    holds, and those against the pool's own writes on the host."""
    g = torch.Generator().manual_seed(4)
    Hq, Hk, D, S, lens, steps = 8, 2, 64, 16, [37, 1, 90], 20
    B, T = len(lens), sum(lens)
    q, k, v, cu = make(lens, Hq, Hk, D, dtype, seed=5)
    pool = FP4KVBlockPool(2, 40, S, Hk, D, device=DEV)
    pool.data.fill_(255)
    tables = torch.randperm(40, generator=g)[:B * 8].view(B, 8).to(DEV)
    place = lambda b, t: tables[b, t // S] * S + t % S
    slots = torch.cat([place(b, torch.arange(n, device=DEV)) for b, n in enumerate(lens)])
    check(hpd.prompt_attention_hip(q, k, v, cu), q, k, v, cu)
    hpd.kv_append_fp4(pool, 1, k, v, slots)
    ctx = torch.tensor(lens, device=DEV)
    twin = FP4KVBlockPool(2, 40, S, Hk, D)
    twin.data.fill_(255)
    for t in range(T):
        twin.write_layer(1, int(slots[t]) // S, int(slots[t]) % S, k[t].cpu(), v[t].cpu())
    for _ in range(steps):
        q1 = torch.randn((B, Hq, D), generator=g).to(dtype).to(DEV)
        k1, v1 = torch.randn((2, B, Hk, D), generator=g).to(dtype).to(DEV)
        new = place(torch.arange(B, device=DEV), ctx)
        hpd.kv_append_fp4(pool, 1, k1, v1, new)
        ctx = ctx + 1
        for b in range(B):
            twin.write_layer(1, int(new[b]) // S, int(new[b]) % S, k1[b].cpu(), v1[b].cpu())
        got = hpd.paged_attention_fp4_hip(q1, pool, tables, ctx, 1)
        for b in range(B):
            n = int(ctx[b])
            kb, vb = (x.double() for x in hpd.kv_gather_fp4(pool, 1, place(b, torch.arange(n, device=DEV))))
            qb = q1[b].double().view(Hk, -1, D) / math.sqrt(D)
            w = torch.softmax(qb @ kb.permute(1, 2, 0).contiguous(), -1)
            X = (qb.abs() @ kb.abs().permute(1, 2, 0).contiguous()).amax(-1).view(Hq, 1)
            want, A = ((w @ x.transpose(0, 1).contiguous()).view(Hq, D) for x in (vb, vb.abs()))
            # As in test_fp4_kv_gpu.py.
            tol = (2 * (D + 4) * U * X + 8 * U + 2 * (n + 32) * U + 2.0 ** -18) * A + torch.finfo(dtype).eps / 2 * want.abs()
            assert ((got[b].double() - want).abs() <= tol).all()
    assert torch.equal(pool.data.cpu(), twin.data)


def exact_scores(power, Hq, Hk, dtype, lens, seed):
    """q, k, v, starts and a scale: scores near 2^power (of e) for two rows of three, a few units
    for the third, every one a sum of two products that f32 holds exactly."""
    q, k, v, cu = make(lens, Hq, Hk, 64, dtype, seed=seed)
    g = torch.Generator().manual_seed(seed)
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    q[..., 0], k[..., 0] = 2.0 ** 15, 2.0 ** 15
    q[..., 1] = 2.0 ** 7  # a step of 2^30 in f32
    q[::3, :, 0] = 0
    k[..., 1] = torch.randint(0, 9, (sum(lens), Hk), generator=g).to(DEV)
    return q, k, v, cu, 2.0 ** (power - 30)


def check_exact_scores(got, q, k, v, cu, scale):
    """Scores have no error here, nor has what they differ by. A weight's exponent is off by 3 u of
    itself (the scale's factor, its product), which moves a weight w = 2^-d by 3 u d w <= 2 u,
    exp2 and the sums as in `tolerance`."""
    out, A, _ = reference(q, k, v, cu, scale)
    half, n = torch.finfo(q.dtype).eps / 2, int((cu[1:] - cu[:-1]).max())
    tol = (16 * U + 2 * (n + 32) * U + 2 * half * (q.dtype != F32)) * A + half * out.abs()
    if q.dtype == F16:
        tol = tol + n * 2.0 ** -38 * float(v.abs().amax()) + 2.0 ** -25
    assert not torch.isnan(got).any()
    off = (got.double() - out).abs()
    assert (off <= tol).all(), f"worst {float((off / tol.clamp_min(1e-300)).max()):.3g} of the tolerance"


@DTYPES
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [4, 12, 15, 16, 18, 20, 22, 24, 27, 30, 34, 60])
def test_scores_of_any_size(power, sign, dtype):
    """Where a score's product with the scale rounds by more than a weight's exponent may."""
    q, k, v, cu, scale = exact_scores(power, 4, 2, dtype, [1, 1, 2, 130, 300], seed=power)
    got = torch.empty(q.shape, dtype=dtype, device=DEV)
    entry(q, k, v, cu, got, sign * scale, 1)
    check_exact_scores(got, q, k, v, cu, sign * scale)


@DTYPES
@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 11, 2.0 ** 13, 2.0 ** 18])
def test_a_row_alone_is_its_value_at_any_score(size, dtype):
    lens, size = [1] * 300, min(size, 2.0 ** 13) if dtype == F16 else size
    q, k, v, cu = make(lens, 2, 1, 64, dtype, seed=11)
    got = hpd.prompt_attention_hip(q * size, k * size, v, cu)
    want = v.expand(-1, 2, -1).double()
    assert ((got.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 4 * U) * want.abs()).all()


@DTYPES
@pytest.mark.parametrize("Hq,Hk,D", [(4, 1, 64), (2, 1, 128), (1, 1, 128), (3, 3, 80), (4, 2, 20)])
def test_a_rows_bits_are_those_of_the_rows_it_sees(Hq, Hk, D, dtype):
    """The same first rows before other ones, which move the others' maxima, hold what is not a
    number, or have scores that are far from 0."""
    lens, same = [333, 41], 100
    q, k, v, cu = make(lens, Hq, Hk, D, dtype, seed=12)
    q = q * 4
    first = hpd.prompt_attention_hip(q, k, v, cu)
    for n in (101, 140, 500):
        for what in ("larger", "far", "nan", "inf"):
            q2, k2, v2, cu2 = make([n, 3], Hq, Hk, D, dtype, seed=13)
            q2, k2, v2 = q2 * 12, k2 * 3, v2 * 2
            for x, y in ((q2, q), (k2, k), (v2, v)):
                x[:same] = y[:same]
            if what == "far":
                q2[same:], k2[same:] = q2[same:] * 2.0 ** 7, k2[same:] * 2.0 ** 7
            elif what != "larger":
                v2[same:, 0, D // 2], k2[same] = float(what), float(what)
            got = hpd.prompt_attention_hip(q2, k2, v2, cu2)
            assert not torch.isnan(got[:same]).any()
            assert torch.equal(got[:same], first[:same]), f"{n} rows, {what}: {int((got[:same] != first[:same]).sum())} values"


@DTYPES
def test_values_near_the_largest_number(dtype):
    """A key somewhat above the running maximum, later: its weight times its value must not
    overflow where the softmax's sum does not."""
    n = 200
    q, k, v = (torch.zeros((n, 1, 64), dtype=dtype, device=DEV) for _ in range(3))
    q[..., 0], k[..., 0] = 8, -30
    k[0, 0, 0], k[40, 0, 0] = 0, 5
    v[:] = 6e4 if dtype == F16 else 2.0 ** 127
    v[..., ::2] *= -1
    check(hpd.prompt_attention_hip(q, k, v, torch.tensor([0, n], device=DEV)), q, k, v, torch.tensor([0, n], device=DEV))


@DTYPES
@pytest.mark.parametrize("scale", [1e-45, -1e-38, 1e20, -1.7e38])
def test_scales_at_the_ends_of_the_range(scale, dtype):
    """Down to scales that make every weight equal, up to ones that leave the largest score alone."""
    scale = torch.tensor(scale, dtype=F32).item()
    q, k, v, cu = make([70, 1, 200], 4, 2, 64, dtype, seed=14)
    if abs(scale) > 1:  # scores without an error
        q, k = q.clone().zero_(), k.clone().zero_()
        q[..., 5], k[..., 5] = 1, torch.arange(len(k), device=DEV)[:, None].remainder(37).to(dtype)
    got = torch.empty(q.shape, dtype=dtype, device=DEV)
    entry(q, k, v, cu, got, scale, 1)
    check_exact_scores(got, q, k, v, cu, scale)
