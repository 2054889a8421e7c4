"""The operators of a request that is served from a 4-bit KV cache, as timed cases.

A program with a 4-bit cache makes these calls per layer: attention of whole prompts,
packed one after the other, over the keys and values as the projection made them
(prompt_attention_hip); the append of those rows to the paged pool in 4 bits
(kv_append_fp4) and their reading back as values (kv_gather_fp4); decode attention over
the pool (paged_attention_fp4_hip).

A head's row of D dims is held in groups of 32 dims (the last one may be shorter): 4-bit
values {0, 0.5, 1, 1.5, 2, 3, 4, 6} and a sign, times one power of two for the group, the
least 2^e (e from -125 to 125) with max |x| <= 7 * 2^e; each element becomes the nearest
value, ties to the even code, 6 at most.

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


def _append(name, T, H, D, S, dtype):
    """T rows of H heads written to the pool in 4 bits; the pool's rows read back."""
    return {"name": name, "op": "append", "T": T, "H": H, "D": D, "S": S, "dtype": dtype}


def _decode(name, B, Hq, Hk, D, S, lo, hi, dtype, lens):
    """B sequences of lo..hi cached tokens, one query token each."""
    return {"name": name, "op": "decode", "B": B, "Hq": Hq, "Hk": Hk, "D": D, "S": S, "lo": lo, "hi": hi,
            "dtype": dtype, "lens": lens}


def _prompt(name, B, Hq, Hk, D, lo, hi, dtype, lens):
    """B prompts of lo..hi tokens, packed."""
    return {"name": name, "op": "prompt", "B": B, "Hq": Hq, "Hk": Hk, "D": D, "lo": lo, "hi": hi, "dtype": dtype,
            "lens": lens}


def listed():
    return [
        # A decode step of four requests of the small fp32 model (8 heads of 32): all launch and latency.
        _append("append_small_model", 4, 8, 32, 16, "f32"),
        # A full decode batch of the decode benchmark's heads.
        _append("append_b256", 256, 32, 128, 16, "bf16"),
        # A packed prefill of grouped heads, odd in length.
        _append("append_prompts", 8191, 8, 128, 32, "f16"),
        # Four requests of the small fp32 model, a few hundred tokens each: where launches and latency count.
        _decode("decode_small_model", 4, 8, 8, 32, 16, 200, 256, "f32", 1),
        # A chat server at light load: 13 conversations of mixed length.
        _decode("decode_chat", 13, 16, 16, 128, 16, 100, 1000, "bf16", 2),
        # The decode benchmark's shape: 64 ragged sequences, 32 heads.
        _decode("decode_batch", 64, 32, 32, 128, 16, 512, 4096, "bf16", 3),
        # A full batch with grouped heads of 64 dims.
        _decode("decode_grouped", 256, 32, 8, 64, 32, 128, 2048, "f16", 4),
        # Long documents, grouped heads: 8 sequences of 32k to 128k tokens.
        _decode("decode_long", 8, 32, 8, 128, 16, 32768, 131072, "bf16", 5),
        # Three short prompts of the small fp32 model.
        _prompt("prompt_small_model", 3, 8, 8, 32, 9, 70, "f32", 6),
        # Two dozen chat prompts of very mixed length, grouped heads.
        _prompt("prompt_chat", 24, 32, 8, 128, 20, 1500, "bf16", 7),
        # Three long documents, grouped heads: the most arithmetic.
        _prompt("prompt_documents", 3, 32, 8, 128, 4000, 8192, "bf16", 8),
        # A mid-sized f16 model's prompts, heads of 80.
        _prompt("prompt_f16", 7, 20, 20, 80, 300, 2100, "f16", 9),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([32, 64, 80, 96, 128, 128])
    S = rng.choice([16, 16, 32, 64])
    while True:
        Hk, G = _log_int(rng, 1, 32), rng.choice([1, 1, 2, 4, 8])
        if Hk * G > 64:
            continue
        if op == "append":
            case = {"op": op, "T": _log_int(rng, 1, 8192), "H": Hk, "D": D, "S": S, "dtype": dtype}
            if work(case)["bytes"] < 5.5e7:
                return case
            continue
        lens = rng.randrange(1 << 20)
        hi = _log_int(rng, 16, 131072) if op == "decode" else _log_int(rng, 8, 8192)
        case = {"op": op, "B": _log_int(rng, 1, 256) if op == "decode" else _log_int(rng, 1, 64), "Hq": Hk * G, "Hk": Hk,
                "D": D, "lo": max(1, hi // rng.choice([1, 2, 8, 32])), "hi": hi, "dtype": dtype, "lens": lens}
        w = work(case)
        if op == "decode":
            case["S"] = S
            if w["bytes"] < 7e8 and w["flops"] < 1.2e10 * (8 if dtype != "f32" else 2):
                return case
        elif w["flops"] < (6e11 if dtype != "f32" else 6e10) and w["bytes"] < 1e9:
            return case


# ------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, dtype, g):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=g)


def _lens(case):
    """Lengths: part of the case (they set its cost), spread over [lo, hi]."""
    r = random.Random(case["lens"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]


def _rows(n, H, D, dtype, channels, g):
    """n tokens' rows: keys differ in size from channel to channel, as projections make them."""
    return (_normal((n, H, D), torch.float32, g) * channels).to(dtype)


def _channels(H, D, g):
    return torch.exp(0.5 * _normal((H, D), torch.float32, g))


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-gpt-inference_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from minivllm import hip_paged_decode
    from minivllm.kv_block_pool import FP4KVBlockPool

    return hip_paged_decode, FP4KVBlockPool


def _pool(N, S, H, D, st, write):
    """An empty 4-bit pool and the function that writes rows into its slots: the framework's, or codes
    [N*S, H, D / 2] (two to a byte) beside scales [N*S, H, groups]. `write` is the plain one."""
    if own:
        hpd, pool = _package()
        st["hpd"], st["pool"] = hpd, pool(1, N, S, H, D, device="cuda")
        st["pool"].data.zero_()
        return lambda k, v, slots: hpd.kv_append_fp4(st["pool"], 0, k, v, slots)
    codes = lambda: torch.zeros((N * S, H, (D + 1) // 2), dtype=torch.uint8, device="cuda")
    scales = lambda: torch.full((N * S, H, -(-D // 32)), 2, dtype=torch.uint8, device="cuda")
    st["kc"], st["vc"], st["ks"], st["vs"] = codes(), codes(), scales(), scales()
    return lambda k, v, slots: write(st, k, v, slots)


def _append_inputs(case, seed, write):
    g, host = _gen(seed), torch.Generator().manual_seed(seed)
    T, H, D, S, dt = case["T"], case["H"], case["D"], case["S"], DTYPES[case["dtype"]]
    N = -(-T // S) + 8
    st = {"case": case}
    put = _pool(N, S, H, D, st, write)
    c = _channels(H, D, g)
    old = _rows(N * S, H, D, dt, c, g)
    with torch.inference_mode():  # what earlier steps left in the pool
        put(old, _normal(old.shape, dt, g), torch.arange(N * S, device="cuda"))
    qkv = _normal((T, 3 * H, D), dt, g)  # one projection's output, q, k and v side by side
    qkv[:, H:2 * H] = (qkv[:, H:2 * H].float() * c).to(dt)
    st["k"], st["v"] = qkv[:, H:2 * H], qkv[:, 2 * H:]
    st["slots"] = torch.randperm(N * S, generator=host)[:T].cuda()
    if T > 256:  # whole prompts: their blocks filled from the front
        order = torch.randperm(N, generator=host)
        st["slots"] = (order[:, None] * S + torch.arange(S)).flatten()[:T].cuda()
    st["all"] = torch.arange(N * S, device="cuda")
    return st


def _decode_inputs(case, seed, write):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    B, Hq, Hk, D, S, lens = case["B"], case["Hq"], case["Hk"], case["D"], case["S"], _lens(case)
    n = [-(-c // S) for c in lens]
    N = sum(n) + 8
    st = {"case": case}
    put = _pool(N, S, Hk, D, st, write)
    perm = torch.randperm(N, generator=torch.Generator().manual_seed(seed))
    tables = torch.full((B, max(n)), -1, dtype=torch.int64)
    at, channels = 0, _channels(Hk, D, g)
    for b, (c, m) in enumerate(zip(lens, n)):
        tables[b, :m] = perm[at:at + m]
        at += m
        slots = (tables[b, :m, None] * S + torch.arange(S)).flatten()[:c].cuda()
        with torch.inference_mode():
            for i in range(0, c, 16384):
                rows = slots[i:i + 16384]
                put(_rows(len(rows), Hk, D, dt, channels, g), _normal((len(rows), Hk, D), dt, g), rows)
    st["q"], st["tables"] = _normal((B, Hq, D), dt, g), tables.cuda()
    st["ctx"] = torch.tensor(lens, dtype=torch.int64).cuda()
    return st


def _prompt_inputs(case, seed):
    g, dt, lens = _gen(seed), DTYPES[case["dtype"]], _lens(case)
    Hq, Hk, D = case["Hq"], case["Hk"], case["D"]
    qkv = _normal((sum(lens), Hq + 2 * Hk, D), dt, g)  # one projection's output, q, k and v side by side
    starts = torch.zeros(len(lens) + 1, dtype=torch.int64)
    starts[1:] = torch.tensor(lens).cumsum(0)
    return {"case": case, "q": qkv[:, :Hq], "k": qkv[:, Hq:Hq + Hk], "v": qkv[:, Hq + Hk:], "starts": starts.cuda()}


def _inputs(case, seed, write):
    if case["op"] == "append":
        return _append_inputs(case, seed, write)
    if case["op"] == "decode":
        return _decode_inputs(case, seed, write)
    return _prompt_inputs(case, seed)


def prepare(case, seed):
    return _inputs(case, seed, _plain_write)


# --------------------------------------------------------------- plain forms

def _grouped(x):
    """[n, H, D] as [n, H, groups, 32], zeros behind the last dim."""
    n, H, D = x.shape
    G = -(-D // 32)
    if D % 32:
        x = torch.cat((x, x.new_zeros((n, H, G * 32 - D))), 2)
    return x.view(n, H, G, 32)


def _encode(rows):
    """Codes (two to a byte, the even dim low) and scale bytes of rows [n, H, D]."""
    x = _grouped(rows.float())
    a = x.abs()
    mantissa, exponent = torch.frexp(a.amax(3))
    e = (exponent - 3 + (mantissa > 0.875).int()).clamp(-125, 125)  # of a maximum of 0: nothing depends on it
    y = torch.ldexp(a, -e[..., None])
    code = torch.zeros_like(y, dtype=torch.uint8)
    for i, border in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += y >= border if i % 2 else y > border  # a tie goes to the even code
    code += torch.signbit(x).to(torch.uint8) * 8
    code = code.flatten(2)[..., :rows.shape[2]]
    if rows.shape[2] % 2:
        code = torch.cat((code, torch.zeros_like(code[..., :1])), 2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _plain_write(st, k, v, slots):
    for x, codes, scales in ((k, "kc", "ks"), (v, "vc", "vs")):
        st[codes][slots], st[scales][slots] = _encode(x)


def _values(codes, scales, D):
    """What codes [n, H, D / 2] and scales [n, H, groups] stand for, in 32 bits."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat((table, -table))
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(2)[..., :D]
    return _scaled(table[both.int()], scales)


def _scaled(x, scales):
    D = x.shape[2]
    factor = torch.ldexp(torch.ones((), device=x.device), scales.int() - 127)
    return (_grouped(x) * factor[..., None]).flatten(2)[..., :D]


def _plain_append(st):
    case = st["case"]
    _plain_write(st, st["k"], st["v"], st["slots"])
    dt, D = DTYPES[case["dtype"]], case["D"]
    return {"k": _values(st["kc"], st["ks"], D).to(dt), "v": _values(st["vc"], st["vs"], D).to(dt)}


def _plain_decode(st):
    case = st["case"]
    B, Hq, Hk, D, S = (case[x] for x in ("B", "Hq", "Hk", "D", "S"))
    q = st["q"].float().view(B, Hk, Hq // Hk, D) / math.sqrt(D)
    out = torch.empty_like(q)
    for b, c in enumerate(_lens(case)):
        slots = (st["tables"][b, :-(-c // S), None] * S + torch.arange(S, device="cuda")).flatten()[:c]
        k, v = (_values(st[x][slots], st[y][slots], D).transpose(0, 1).contiguous()
                for x, y in (("kc", "ks"), ("vc", "vs")))  # [Hk, c, D]
        s = q[b] @ k.transpose(1, 2)
        p = torch.exp(s - s.amax(2, keepdim=True))
        out[b] = (p @ v) / p.sum(2, keepdim=True)
    return out.view(B, Hq, D).to(st["q"].dtype)


def _plain_prompt(st):
    case = st["case"]
    Hq, Hk, D = case["Hq"], case["Hk"], case["D"]
    G, out, at = Hq // Hk, torch.empty(st["q"].shape, dtype=st["q"].dtype, device="cuda"), 0
    for n in _lens(case):
        q, k, v = (st[x][at:at + n].float().transpose(0, 1).contiguous() for x in ("q", "k", "v"))
        for lo in range(0, n, 1024):
            hi = min(n, lo + 1024)
            s = (q[:, lo:hi].reshape(Hk, G * (hi - lo), D) @ k[:, :hi].transpose(1, 2)) / math.sqrt(D)
            s = s.view(Hk, G, hi - lo, hi)
            later = torch.arange(hi, device="cuda")[None] > torch.arange(lo, hi, device="cuda")[:, None]
            s = s.masked_fill(later, -math.inf)
            p = torch.exp(s - s.amax(3, keepdim=True))
            total = p.sum(3, keepdim=True)
            o = (p.view(Hk, G * (hi - lo), hi) @ v[:, :hi]).view(Hk, G, hi - lo, D) / total
            out[at + lo:at + hi] = o.view(Hq, hi - lo, D).transpose(0, 1).to(out.dtype)
        at += n
    return out


def run(st):
    case = st["case"]
    with torch.inference_mode():
        if not own:
            return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt}[case["op"]](st)
        hpd = _package()[0]
        if case["op"] == "prompt":
            return hpd.prompt_attention_hip(st["q"], st["k"], st["v"], st["starts"])
        if case["op"] == "decode":
            return hpd.paged_attention_fp4_hip(st["q"], st["pool"], st["tables"], st["ctx"], 0)
        hpd.kv_append_fp4(st["pool"], 0, st["k"], st["v"], st["slots"])
        k, v = hpd.kv_gather_fp4(st["pool"], 0, st["all"], dtype=DTYPES[case["dtype"]])
        return {"k": k, "v": v}


# ------------------------------------------------------------------ in 64 bits

def _held64(rows):
    """What rows [n, H, D] are held as: by the size of a step around each element, in 64 bits."""
    n, H, D = rows.shape
    out = torch.empty(rows.shape, dtype=torch.float64, device=rows.device)
    for d in range(0, D, 32):
        x = rows[:, :, d:d + 32].double()
        top = x.abs().amax(2, keepdim=True)
        e = torch.ceil(torch.log2(top / 7)).clamp(-125, 125)
        e = torch.where(7 * torch.exp2(e - 1) >= top, e - 1, e)  # where the logarithm fell on the far side
        e = torch.where(7 * torch.exp2(e) < top, e + 1, e).clamp(-125, 125)
        unit = torch.exp2(e)
        y = x / unit
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(1, 8)))) / 2
        out[:, :, d:d + 32] = (torch.round(y / step) * step).clamp(-6, 6) * unit
    return out


def _write64(st, k, v, slots):
    if "k64" not in st:
        st["k64"], st["v64"] = (torch.zeros(st["kc"].shape[:2] + k.shape[2:], dtype=torch.float64, device="cuda")
                                for _ in range(2))
    st["k64"][slots], st["v64"][slots] = _held64(k), _held64(v)


def _attend64(q, k, v, allowed=None):
    """q [n, Hq, D] over k, v [m, Hk, D], one head after the other."""
    G, out = q.shape[1] // k.shape[1], torch.empty(q.shape, dtype=torch.float64, device="cuda")
    for h in range(q.shape[1]):
        kh, vh = (x[:, h // G].double().contiguous() for x in (k, v))
        s = q[:, h].double() @ kh.t().contiguous() / math.sqrt(q.shape[2])
        if allowed is not None:
            s = s.masked_fill(~allowed, -math.inf)
        out[:, h] = torch.softmax(s, 1) @ vh
    return out


def exact(case, seed):
    global own
    framework, own = own, False  # the inputs alone, without the framework's pool
    try:
        st = _inputs(case, seed, _write64)
    finally:
        own = framework
    with torch.inference_mode():
        if case["op"] == "append":
            _write64(st, st["k"], st["v"], st["slots"])
            return {"k": st["k64"], "v": st["v64"]}
        if case["op"] == "decode":
            out, S = [], case["S"]
            for b, c in enumerate(_lens(case)):
                slots = (st["tables"][b, :-(-c // S), None] * S + torch.arange(S, device="cuda")).flatten()[:c]
                out.append(_attend64(st["q"][b:b + 1], st["k64"][slots], st["v64"][slots]))
            return torch.cat(out)
        out, at = [], 0
        for n in _lens(case):
            q, k, v = (st[x][at:at + n] for x in ("q", "k", "v"))
            out.append(_attend64(q, k, v, torch.ones((n, n), dtype=torch.bool, device="cuda").tril()))
            at += n
        return torch.cat(out)


# ------------------------------------------------------------------------ work

def work(case):
    D, e = case["D"], EB[case["dtype"]]
    held = -(-D // 2) + -(-D // 32)  # bytes of a head's row in 4 bits
    if case["op"] == "append":
        T, H, S = case["T"], case["H"], case["S"]
        rows = (-(-T // S) + 8) * S
        # The new rows read and written, then the pool's rows read and their values written.
        return {"bytes": 2 * H * (T * (e * D + held) + rows * (held + e * D)) + 8 * (T + rows),
                "flops": 2 * H * D * (3 * T + rows)}
    Hq, Hk, lens = case["Hq"], case["Hk"], _lens(case)
    if case["op"] == "decode":
        blocks = sum(-(-c // case.get("S", 16)) for c in lens)
        return {"bytes": 2 * Hk * held * sum(lens) + 2 * e * len(lens) * Hq * D + 8 * (blocks + len(lens)),
                "flops": 4 * Hq * D * sum(lens)}
    return {"bytes": 2 * e * sum(lens) * D * (Hq + Hk) + 8 * (len(lens) + 1),
            "flops": 4 * Hq * D * sum(n * (n + 1) // 2 for n in lens)}
