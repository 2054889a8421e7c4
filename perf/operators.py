"""The operators of a rotary decode or prefill step, as timed cases.

Three calls of a serving program, per layer: the norms of the query and key heads
with the position rotation (qk_norm_rope_hip), the append of keys and values to
the paged pool with the same rotation on the way (kv_append_rope_hip), and decode
attention of a batch whose sequences begin with the same cached blocks
(paged_attention_shared_prefix_hip).

  own = False   run() computes the plain form, elementary torch operations in 32
                bits; True: the framework's calls
  listed()  the named cases;  draw(rng)  another case of the same ranges;
  prepare(case, seed)  what a program holds before the call, on the GPU;
  run(state)  one pass;  exact(case, seed)  the same outputs in 64 bits;
  work(case)  what a pass cannot do without.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EB = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
BASE = 10000.0


def _rope(name, op, T, Hq, Hk, D, R, dtype, interleaved, norm, far):
    """One rope case: T rows of Hq query and Hk key heads, R of D dims rotated, positions below `far`."""
    return {"name": name, "op": op, "T": T, "Hq": Hq, "Hk": Hk, "D": D, "R": R, "dtype": dtype,
            "interleaved": interleaved, "norm": norm, "far": far, "S": 16}


def _shared(name, B, Hq, Hk, D, S, shared, lo, hi, dtype, lens):
    """B sequences that share `shared` blocks of S tokens and go on for lo..hi tokens of their own."""
    return {"name": name, "op": "shared", "B": B, "Hq": Hq, "Hk": Hk, "D": D, "S": S, "shared": shared, "lo": lo,
            "hi": hi, "dtype": dtype, "lens": lens}


def listed():
    return [
        # One token of the small fp32 model (8 heads of 32): the smallest call, all launch and latency.
        _rope("norm_rope_token", "norm_rope", 1, 8, 8, 32, 32, "f32", False, True, 2048),
        # A short prompt's chunk of an odd length, adjacent pairs rotated.
        _rope("norm_rope_chunk", "norm_rope", 203, 16, 16, 128, 128, "bf16", True, True, 8192),
        # A long prompt in one pass, grouped heads.
        _rope("norm_rope_prompt", "norm_rope", 8192, 32, 8, 128, 128, "bf16", False, True, 32768),
        # A decode step of 13 conversations, rotation only.
        _rope("append_rope_chat", "append", 13, 16, 16, 128, 128, "bf16", False, False, 8192),
        # A full decode batch, head norms and rotation on the way into the pool.
        _rope("append_rope_b256", "append", 256, 32, 32, 128, 128, "bf16", False, True, 131072),
        # A full-budget prefill chunk with grouped heads, half of each head rotated.
        _rope("append_rope_chunk", "append", 2048, 32, 8, 128, 64, "f16", True, True, 32768),
        # Four requests of the small fp32 model on one short prompt: where launches and latency count.
        _shared("shared_small_model", 4, 8, 8, 32, 16, 8, 72, 128, "f32", 7),
        # A chat server at light load: 13 conversations under one system prompt.
        _shared("shared_chat", 13, 16, 16, 128, 16, 50, 20, 500, "bf16", 8),
        # The decode benchmark's batch and heads, 4096 tokens of common prompt before ragged turns.
        _shared("shared_batch", 64, 32, 32, 128, 16, 256, 64, 1024, "bf16", 9),
        # 128 short questions about one long document, grouped heads: the most arithmetic per byte.
        _shared("shared_document", 128, 32, 8, 128, 16, 4096, 32, 256, "bf16", 10),
        # One GPU's share of a head split: 8 query heads on one KV head, f16, long turns.
        _shared("shared_head_share", 64, 8, 1, 128, 32, 250, 50, 3000, "f16", 11),
        # A mid-sized fp32 model, two dozen sequences.
        _shared("shared_f32", 24, 12, 12, 64, 16, 94, 16, 400, "f32", 12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([32, 64, 80, 96, 128, 128])
    if rng.random() < 0.5:
        while True:
            Hk, G = _log_int(rng, 1, 32), rng.choice([1, 1, 2, 4, 8])
            T, far = _log_int(rng, 1, 8192), _log_int(rng, 256, 131072)
            R = rng.choice([D, D, D // 2])
            op = rng.choice(["norm_rope", "append"])
            case = {"op": op, "T": T, "Hq": Hk * G, "Hk": Hk, "D": D, "R": R, "dtype": dtype,
                    "interleaved": rng.random() < 0.4, "norm": op == "norm_rope" or rng.random() < 0.5, "far": far,
                    "S": rng.choice([16, 16, 32, 64])}
            if Hk * G <= 64 and work(case)["bytes"] < 2.4e8:
                return case
    while True:
        Hk, G = _log_int(rng, 1, 32), rng.choice([1, 1, 2, 4, 8])
        B, S = _log_int(rng, 2, 256), rng.choice([16, 16, 32, 64])
        shared, hi = max(1, _log_int(rng, 64, 65536) // S), _log_int(rng, 16, 3000)
        case = {"op": "shared", "B": B, "Hq": Hk * G, "Hk": Hk, "D": D, "S": S, "shared": shared,
                "lo": max(1, hi // rng.choice([1, 2, 8, 32])), "hi": hi, "dtype": dtype, "lens": rng.randrange(1 << 20)}
        w = work(case)
        # At most about what the largest listed case takes at 6 TB/s and the matrix cores' rates.
        if Hk * G <= 64 and w["bytes"] / 6e12 + w["flops"] / (1e15 if dtype != "f32" else 1.2e14) < 1.9e-4:
            return case


# ------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, dtype, g):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=g)


def _lens(case):
    """Own tokens of each sequence: part of the case (they set its cost), spread over [lo, hi]."""
    r = random.Random(case["lens"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]


def _table(case):
    """cos and sin of every position's angles, [far, R] f32, from angles in 64 bits."""
    half = case["R"] // 2
    freq = BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = torch.arange(case["far"], dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _rope_inputs(case, seed):
    g, host, dt = _gen(seed), torch.Generator().manual_seed(seed), DTYPES[case["dtype"]]
    T, Hq, Hk, D, S = (case[x] for x in ("T", "Hq", "Hk", "D", "S"))
    qkv = _normal((T, Hq + 2 * Hk, D), dt, g)  # one projection's output, q, k and v side by side
    st = {"q": qkv[:, :Hq], "k": qkv[:, Hq:Hq + Hk], "v": qkv[:, Hq + Hk:], "table": _table(case)}
    start = int(torch.randint(0, max(1, case["far"] - T), (), generator=host))
    if T <= 256:  # a decode batch: each row a sequence's next token
        st["positions"] = torch.randint(0, case["far"], (T,), generator=host).cuda()
    else:  # a chunk of one prompt
        st["positions"] = torch.arange(start, start + T).remainder(case["far"]).cuda()
    st["qw"] = st["kw"] = None
    if case["norm"]:
        st["qw"], st["kw"] = (1 + 0.1 * _normal((D,), torch.float32, g).to(dt) for _ in range(2))
    if case["op"] == "append":
        n = -(-T // S) + 8
        st["slots"] = torch.randperm(n * S, generator=host)[:T].cuda()
        st["kp"], st["vp"] = (_normal((1, n, S, Hk, D), dt, g) for _ in range(2))
    return st


def _shared_inputs(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    B, Hq, Hk, D, S, P = (case[x] for x in ("B", "Hq", "Hk", "D", "S", "shared"))
    lens = _lens(case)
    n = [-(-c // S) for c in lens]
    N = P + sum(n) + 8
    perm = torch.randperm(N, generator=torch.Generator().manual_seed(seed))
    tables = torch.full((B, P + max(n)), -1, dtype=torch.int64)
    tables[:, :P] = perm[:P]
    at = P
    for b, k in enumerate(n):
        tables[b, P:P + k] = perm[at:at + k]
        at += k
    ctx = torch.tensor([P * S + c for c in lens], dtype=torch.int64)
    st = {"q": _normal((B, Hq, D), dt, g), "tables": tables.cuda(), "ctx": ctx.cuda()}
    st["kp"], st["vp"] = (_normal((1, N, S, Hk, D), dt, g) for _ in range(2))
    return st


def _inputs(case, seed):
    return _shared_inputs(case, seed) if case["op"] == "shared" else _rope_inputs(case, seed)


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-gpt-inference_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from minivllm import hip_paged_decode
    from minivllm.kv_block_pool import KVBlockPool

    return hip_paged_decode, KVBlockPool


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:
        st["hpd"], pool = _package()
        if "kp" in st:
            _, n, S, H, D = st["kp"].shape
            st["pool"] = pool(1, n, S, H, D, device="cuda", dtype=st["kp"].dtype)
            st["pool"].k.copy_(st.pop("kp"))
            st["pool"].v.copy_(st.pop("vp"))
    return st


# --------------------------------------------------------------- plain forms

def _rotated(x, w, rows, case):
    """The head norm (with w) and the rotation by the table's rows, in 32 bits."""
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
    R = case["R"]
    cos, sin = rows[:, None, :R // 2], rows[:, None, R // 2:]
    out = y.clone()
    if case["interleaved"]:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        out[..., 0:R:2], out[..., 1:R:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., :R // 2], y[..., R // 2:R]
        out[..., :R // 2], out[..., R // 2:R] = a * cos - b * sin, b * cos + a * sin
    return out.to(x.dtype)


def _plain_rope(st):
    case = st["case"]
    rows = st["table"][st["positions"]]
    q, k = _rotated(st["q"], st["qw"], rows, case), _rotated(st["k"], st["kw"], rows, case)
    if case["op"] == "norm_rope":
        return {"q": q, "k": k}
    S = case["S"]
    blocks, offsets = torch.div(st["slots"], S, rounding_mode="floor"), st["slots"] % S
    st["kp"][0, blocks, offsets] = k
    st["vp"][0, blocks, offsets] = st["v"]
    return {"q": q, "k_pool": st["kp"], "v_pool": st["vp"]}


def _plain_shared(st):
    case = st["case"]
    B, Hq, Hk, D, S, P = (case[x] for x in ("B", "Hq", "Hk", "D", "S", "shared"))
    G, ctx, tables = Hq // Hk, st["ctx"], st["tables"]
    q = st["q"].view(B, Hk, G, D).transpose(0, 1).float() / math.sqrt(D)  # [Hk, B, G, D]
    # The shared keys once for all rows: [Hk, P S, D] in 32 bits.
    k, v = (t[0][tables[0, :P]].flatten(0, 1).transpose(0, 1).float().contiguous() for t in (st["kp"], st["vp"]))
    s = q.reshape(Hk, B * G, D) @ k.transpose(1, 2).contiguous()
    # Each row's own keys, padded to the longest row: [B Hk, n S, D].
    own_tables = tables[:, P:]
    n = own_tables.shape[1]
    ok, ov = (t[0][own_tables.clamp_min(0)].flatten(1, 2).transpose(1, 2).float().contiguous()
              .view(B * Hk, n * S, D) for t in (st["kp"], st["vp"]))
    past = torch.arange(n * S, device=ctx.device)[None] >= (ctx - P * S)[:, None]
    so = (q.transpose(0, 1).reshape(B * Hk, G, D) @ ok.transpose(1, 2).contiguous()).view(B, Hk, G, n * S)
    so = so.masked_fill(past[:, None, None], -math.inf)
    s = s.view(Hk, B, G, P * S).transpose(0, 1)  # [B, Hk, G, P S]
    m = torch.maximum(s.amax(-1), so.amax(-1))[..., None]
    p, po = torch.exp(s - m), torch.exp(so - m)
    total = p.sum(-1, keepdim=True) + po.sum(-1, keepdim=True)
    out = (p.transpose(0, 1).reshape(Hk, B * G, P * S) @ v).view(Hk, B, G, D).transpose(0, 1)
    out = out + (po.reshape(B * Hk, G, n * S) @ ov).view(B, Hk, G, D)
    return (out / total).reshape(B, Hq, D).to(st["q"].dtype)


def run(st):
    case = st["case"]
    with torch.inference_mode():
        if not own:
            return _plain_shared(st) if case["op"] == "shared" else _plain_rope(st)
        hpd = st["hpd"]
        if case["op"] == "shared":
            return hpd.paged_attention_shared_prefix_hip(st["q"], st["pool"], st["tables"], st["ctx"], 0,
                                                         shared_blocks=case["shared"])
        if case["op"] == "norm_rope":
            q, k = hpd.qk_norm_rope_hip(st["q"], st["k"], st["positions"], st["table"], st["qw"], st["kw"], eps=EPS,
                                        interleaved=case["interleaved"])
            return {"q": q, "k": k}
        q = hpd.kv_append_rope_hip(st["pool"], 0, st["q"], st["k"], st["v"], st["slots"], st["positions"],
                                   st["table"], st["qw"], st["kw"], eps=EPS, interleaved=case["interleaved"])
        return {"q": q, "k_pool": st["pool"].k, "v_pool": st["pool"].v}


# ------------------------------------------------------------------ in 64 bits

def _turned64(x, w, rows, case):
    """Norm and rotation as a complex product: pair j times e^(i angle)."""
    x = x.double()
    if w is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    R, half = case["R"], case["R"] // 2
    order = torch.arange(R, device=x.device)
    pairs = order.view(half, 2) if case["interleaved"] else order.view(2, half).t()
    turn = torch.complex(rows[:, :half].double(), rows[:, half:].double())
    z = torch.view_as_complex(x[..., pairs].contiguous()) * turn[:, None]
    x = x.clone()
    x[..., pairs] = torch.view_as_real(z)
    return x


def _shared64(case, st):
    B, Hq, Hk, D, S, P = (case[x] for x in ("B", "Hq", "Hk", "D", "S", "shared"))
    G, out = Hq // Hk, torch.empty((B, Hq, D), dtype=torch.float64, device="cuda")
    lens = _lens(case)
    prefix = st["tables"][0, :P]
    for h in range(Hk):
        k, v = (t[0, :, :, h][prefix].reshape(P * S, D).double() for t in (st["kp"], st["vp"]))
        q = st["q"][:, h * G:(h + 1) * G].double() / math.sqrt(D)
        shared = (q.reshape(B * G, D) @ k.t().contiguous()).view(B, G, P * S)
        for b, c in enumerate(lens):
            mine = st["tables"][b, P:P + -(-c // S)]
            kb, vb = (t[0, :, :, h][mine].reshape(-1, D)[:c].double() for t in (st["kp"], st["vp"]))
            p = torch.softmax(torch.cat((shared[b], q[b] @ kb.t().contiguous()), 1), 1)
            out[b, h * G:(h + 1) * G] = p[:, :P * S].contiguous() @ v + p[:, P * S:].contiguous() @ vb
    return out


def exact(case, seed):
    st = _inputs(case, seed)
    with torch.inference_mode():
        if case["op"] == "shared":
            return _shared64(case, st)
        rows = st["table"].index_select(0, st["positions"])
        q, k = _turned64(st["q"], st["qw"], rows, case), _turned64(st["k"], st["kw"], rows, case)
        if case["op"] == "norm_rope":
            return {"q": q, "k": k}
        kp, vp = st["kp"].double(), st["vp"].double()
        kp[0].view(-1, case["Hk"], case["D"])[st["slots"]] = k
        vp[0].view(-1, case["Hk"], case["D"])[st["slots"]] = st["v"].double()
        return {"q": q, "k_pool": kp, "v_pool": vp}


# ------------------------------------------------------------------------ work

def work(case):
    Hq, Hk, D, e = case["Hq"], case["Hk"], case["D"], EB[case["dtype"]]
    if case["op"] == "shared":
        B, S, P, lens = case["B"], case["S"], case["shared"], _lens(case)
        tokens = sum(lens)
        blocks = P + sum(-(-c // S) for c in lens)
        return {"bytes": 2 * e * Hk * D * (P * S + tokens) + 2 * e * B * Hq * D + 8 * (blocks + B),
                "flops": 4 * Hq * D * (B * P * S + tokens)}
    T, R = case["T"], case["R"]
    rotated, values = Hq + Hk, Hk if case["op"] == "append" else 0
    return {"bytes": 2 * e * T * D * (rotated + values) + 4 * R * min(T, case["far"]) + 8 * T * (2 if values else 1)
            + (2 * e * D if case["norm"] else 0),
            "flops": T * rotated * (3 * R + (4 * D if case["norm"] else 0))}
