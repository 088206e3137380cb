"""Three operators of the layer-stack models, as cases that can be timed and checked.

* `rotate` (tbl_head_rotation_forward): RMS norm of every query and key head and the rotation by its position, in one pass over
  stacked projections;
* `cache4` (tbl_quantized_forward, tbl_quantized_read): grouped attention over a cache that holds keys and values in 4 bits.  A call norms,
  rotates, rounds and appends its tokens, attends, and gates;
* `decay` (tbl_decay_forward): linear attention with a decay for each head, normed, rotated, read out, normed and gated.

All three take the fp32 projections of a step of n_seq sequences of n_tok tokens, as the linear layers of the package leave them.

A row of the 4-bit cache, [slot][kv head][token]: codes of the key (two numbers a byte, the even dimension in the low half), codes of the value,
then one scale byte for every 16 numbers of the key, then of the value; head sizes are padded with zeros to a multiple of 64, rows to 16 bytes.  A number is
code (e2m1) x scale (e4m3) x the layer's fp32 scale of keys or of values.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
BASE = 10000.0
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def rotate(dtype, seqs, tokens, q_heads, k_heads, dim, rot_dim, interleaved, start):
    return {"op": "rotate", "dtype": dtype, "seqs": seqs, "tokens": tokens, "heads": q_heads, "kv_heads": k_heads, "dim": dim, "rot_dim": rot_dim,
            "interleaved": interleaved, "context": start + tokens}


def cache4(dtype, seqs, tokens, context, heads, kv_heads, dim, rot_dim, interleaved=False, gated=True):
    return {"op": "cache4", "dtype": dtype, "seqs": seqs, "tokens": tokens, "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot_dim": rot_dim, "interleaved": interleaved, "gated": gated}


def decay(dtype, seqs, tokens, heads, dim, rot_dim, start, interleaved=False, gated=True):
    return {"op": "decay", "dtype": dtype, "seqs": seqs, "tokens": tokens, "context": start + tokens, "heads": heads, "kv_heads": heads, "dim": dim,
            "rot_dim": rot_dim, "interleaved": interleaved, "gated": gated}


def listed():
    return [
        # one token of one user: latency
        {"name": "rotate_token", **rotate("bfloat16", 1, 1, 32, 8, 128, 128, False, 700)},
        # a portion of a long prompt: bandwidth
        {"name": "rotate_prompt", **rotate("bfloat16", 1, 8192, 32, 8, 128, 128, False, 0)},
        # several ragged prompts side by side in fp32, heads that fit no vector, pairs of neighbours, a part of the head rotated
        {"name": "rotate_ragged", **rotate("float32", 7, 333, 12, 4, 90, 44, True, 51)},
        # one user of a chat with some history
        {"name": "cache4_token", **cache4("bfloat16", 1, 1, 900, 32, 8, 128, 128)},
        # many users at once, each with a history of their own length
        {"name": "cache4_batch", **cache4("bfloat16", 64, 1, 4096, 32, 8, 128, 128)},
        # a question about a very long document, token by token
        {"name": "cache4_document", **cache4("bfloat16", 1, 1, 131001, 32, 8, 128, 64)},
        # a portion of a prompt behind a long history
        {"name": "cache4_prompt", **cache4("bfloat16", 1, 2048, 8192, 32, 8, 128, 128)},
        # the check of a few drafted tokens of some users in fp32, odd sizes
        {"name": "cache4_ragged", **cache4("float32", 5, 3, 777, 10, 2, 90, 44, True, False)},
        # one token of one user: latency
        {"name": "decay_token", **decay("bfloat16", 1, 1, 32, 128, 128, 700)},
        # many users at once: the states' bytes
        {"name": "decay_batch", **decay("bfloat16", 64, 1, 32, 128, 128, 900)},
        # a long prompt
        {"name": "decay_prompt", **decay("bfloat16", 1, 8192, 32, 128, 128, 0)},
        # short prompts side by side in fp32, odd sizes
        {"name": "decay_ragged", **decay("float32", 3, 301, 10, 90, 44, 17, True, False)},
    ]


def spread(rng, low, high):
    """A whole number whose logarithm is spread evenly."""
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(("rotate", "cache4", "cache4", "cache4", "decay", "decay", "decay"))
    dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
    dim = rng.choice((64, 64, 128, 128, 128, 2 * rng.randint(16, 64), 2 * rng.randint(16, 128)))
    rot = rng.choice((0, dim, dim, 2 * rng.randint(1, dim // 2)))
    pairs, gated = rng.random() < 0.3, rng.random() < 0.7
    if op == "rotate":
        rows = spread(rng, 1, 8192)
        seqs = spread(rng, 1, min(rows, 64))
        kv = rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 2, 4))
        tokens = max(1, min(rows, (8192 * 5120) // ((heads + kv) * dim)) // seqs)
        return rotate(dtype, seqs, tokens, heads, kv, dim, rot, pairs, rng.randint(0, 2000))
    if op == "cache4":
        kv = rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 2, 4, 4, 6, 8))
        fp32 = dtype == "float32"
        kind = rng.choice(("one", "one", "few", "prompt"))
        if kind == "one":                                      # cached tokens of all sequences and heads
            seqs = spread(rng, 1, 8 if fp32 else 64)
            return cache4(dtype, seqs, 1, spread(rng, 1, min(131000, (1 << (24 if fp32 else 28)) // (seqs * kv * dim))), heads, kv, dim, rot, pairs, gated)
        if kind == "few":
            seqs, tokens = spread(rng, 1, 8), rng.randint(2, 24)
            return cache4(dtype, seqs, tokens, tokens + spread(rng, 1, (1 << (21 if fp32 else 25)) // (seqs * kv * dim)), heads, kv, dim, rot, pairs, gated)
        tokens = min(spread(rng, 40, 200 if fp32 else 2048), (2048 * 4096) // (heads * dim))
        return cache4(dtype, 1, tokens, tokens + rng.choice((0, spread(rng, 1, 500 if fp32 else 6000))), heads, kv, dim, rot, pairs, gated)
    heads = spread(rng, 1, 32)
    kind = rng.choice(("one", "few", "prompt", "prompt"))
    if kind == "one":
        return decay(dtype, spread(rng, 1, min(64, (1 << 25) // (heads * dim * dim))), 1, heads, dim, rot, rng.randint(0, 2000), pairs, gated)
    if kind == "few":
        return decay(dtype, spread(rng, 1, 16), rng.randint(2, 40), heads, dim, rot, rng.randint(0, 2000), pairs, gated)
    rows = spread(rng, 64, 400 if dtype == "float32" else min(8192, (8192 * 4096) // (heads * dim)))
    seqs = spread(rng, 1, min(4, rows // 16))
    return decay(dtype, seqs, rows // seqs, heads, dim, rot, rng.randint(0, 2000), pairs, gated)


# ---- sizes ------------------------------------------------------------------------------------------------------------------
def starts(case):
    """Tokens that every sequence holds before the call: the first one the most, the others up to a third fewer."""
    most = case["context"] - case["tokens"]
    return [most - (i * 37) % (most // 3 + 1) for i in range(case["seqs"])]


def padded(n, to=64):
    return (n + to - 1) // to * to


def row_bytes(case):
    n = padded(case["dim"])
    return padded(n + n // 8, 16)


def columns(case):
    """Columns of the stacked projections: queries, keys, values, gate."""
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    return (h * d, g * d, 0 if case["op"] == "rotate" else g * d, h * d if case.get("gated") else 0)


def work(case):
    rows, d, h, g = case["seqs"] * case["tokens"], case["dim"], case["heads"], case["kv_heads"]
    size = 2 if case["dtype"] == "bfloat16" else 4
    read = 4 * rows * sum(columns(case))
    turned = 6 * rows * (h + g) * d
    tables = 4 * case["rot_dim"] * min(rows, case["context"])
    if case["op"] == "rotate":
        return {"bytes": read + tables + size * rows * (h + g) * d, "flops": turned}
    out = size * rows * h * d
    if case["op"] == "cache4":
        token = d + 2 * ((d + 15) // 16)                       # codes and scales of a key and a value
        cached = g * token * sum(s + case["tokens"] for s in starts(case)) + 2 * 4 * rows * g * d
        seen = sum(case["tokens"] * s + case["tokens"] * (case["tokens"] + 1) // 2 for s in starts(case))
        return {"bytes": read + tables + out + cached, "flops": turned + 4 * h * d * seen}
    return {"bytes": read + tables + out + 2 * 4 * case["seqs"] * h * d * d, "flops": turned + 4 * rows * h * d * d}


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def rounded4(x, unit):
    """Codes 0 .. 15 and scales (e4m3) of groups of 16 numbers in units of `unit` (fp32 on the device); x fp32 [..., multiple of 16]."""
    x = x.unflatten(-1, (-1, 16))
    six, most = x.new_tensor(6.0), x.abs().amax(-1)
    scale = (most / (unit * six)).clamp(max=448.0).to(torch.float8_e4m3fn)
    y = x / (scale.float() * unit).unsqueeze(-1)
    a = y.abs()
    code = (a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int()
    code = torch.where(scale.float().unsqueeze(-1) > 0, code + 8 * (x < 0).int(), 0)
    return code.flatten(-2), scale


def cached_rows(keys, values, units, size):
    """Bytes of cache rows; keys, values fp32 [..., padded head size]."""
    (kc, ks), (vc, vs) = rounded4(keys, units[0]), rounded4(values, units[1])
    both = lambda c: (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
    row = torch.cat([both(kc), both(vc), ks.view(torch.uint8), vs.view(torch.uint8)], -1)
    return torch.nn.functional.pad(row, (0, size - row.shape[-1]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    seqs, tokens, d, h, g = case["seqs"], case["tokens"], case["dim"], case["heads"], case["kv_heads"]
    rows, capacity = seqs * tokens, padded(case["context"], 16)
    dtype = getattr(torch, case["dtype"])
    s = {"case": case, "dtype": dtype, "capacity": capacity, "proj": rand(rows, sum(columns(case))),
         "slots": torch.randperm(seqs, generator=gen, device="cuda").int()}
    begin = torch.tensor(starts(case), device="cuda", dtype=torch.int32)
    s["positions"] = torch.empty_like(begin)
    s["positions"][s["slots"].long()] = begin
    half = case["rot_dim"] // 2
    angles = torch.arange(capacity, device="cuda", dtype=torch.float64)[:, None] * BASE ** (-torch.arange(half, device="cuda", dtype=torch.float64) / max(half, 1))
    s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
    s["q_norm"], s["k_norm"] = 1.0 + 0.1 * rand(d), 1.0 + 0.1 * rand(d)
    if case["op"] == "rotate":
        s["q"], s["k"] = torch.empty(rows, h, d, dtype=dtype, device="cuda"), torch.empty(rows, g, d, dtype=dtype, device="cuda")
        return s
    s["out"], s["scale"] = torch.empty(rows, h * d, dtype=dtype, device="cuda"), d ** -0.5
    if case["op"] == "cache4":
        # keys have been normed, values have the spread of a projection; the rows behind a sequence hold what an earlier one left there
        s["units"] = torch.tensor([0.02, 0.03], device="cuda")
        n, size = padded(d), row_bytes(case)
        s["cache"] = torch.empty(seqs, g, capacity, size, dtype=torch.uint8, device="cuda")
        some = max(1, (1 << 25) // (g * n))
        for slot in range(seqs):
            for lo in range(0, capacity, some):
                part = [torch.nn.functional.pad(rand(g, min(some, capacity - lo), d), (0, n - d)) for _ in range(2)]
                s["cache"][slot, :, lo:lo + some] = cached_rows(*part, s["units"], size)
        s["keys"], s["values"] = (torch.empty(rows, g, d, device="cuda") for _ in range(2))
        return s
    # decays from a few tokens' memory to a few thousands'
    s["log_decay"] = -torch.exp2(-1.0 - 10.0 * torch.rand(h, generator=gen, device="cuda"))
    s["norm"] = 1.0 + 0.1 * rand(h * d)
    s["states"], s["next"] = rand(seqs, h, d, d), torch.zeros(seqs, h, d, d, device="cuda")
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------------------
def plan_of(s):
    """Descriptors, workspace and arguments, which a program keeps beside its weights."""
    import ctypes as C

    from reimagined_b200 import capi
    c, lib = s["case"], capi.stack_lib()
    precision = capi.BF16 if s["dtype"] == torch.bfloat16 else capi.F32
    p = lambda name: s[name].data_ptr()
    rot = capi.HeadRotation(p("q_norm"), p("k_norm"), p("cos"), p("sin"), c["rot_dim"], s["capacity"], int(c["interleaved"]))
    where = (p("slots"), p("positions"), c["seqs"], c["tokens"])
    if c["op"] == "rotate":
        args = (C.byref(rot), precision, EPS, p("proj"), s["proj"].shape[1], c["heads"], c["kv_heads"], c["dim"], *where, p("q"), p("k"))
        return [(lib.tbl_head_rotation_forward, args)], (s["q"], s["k"]), (rot, lib, capi)
    dense = capi.DenseView(s["proj"].data_ptr(), None, c["heads"] * c["dim"], sum(columns(c)))
    back = capi.DenseView(s["proj"].data_ptr(), None, c["heads"] * c["dim"], c["heads"] * c["dim"])
    if c["op"] == "cache4":
        units = s["units"].tolist()
        m = capi.QuantizedMixer(dense, back, rot, c["heads"], c["kv_heads"], c["dim"], int(c["gated"]), s["scale"], units[0], units[1])
        need = lib.tbl_quantized_workspace_bytes(C.byref(m), precision, 0, c["seqs"], c["tokens"], c["context"])
        space = torch.empty(need, dtype=torch.uint8, device="cuda")
        cache = (p("cache"), c["seqs"], s["capacity"])
        calls = [(lib.tbl_quantized_forward, (C.byref(m), precision, 0, EPS, p("proj"), *cache, *where, c["context"], p("out"), space.data_ptr(), need)),
                 (lib.tbl_quantized_read, (C.byref(m), capi.F32, *cache, *where, p("keys"), p("values")))]
        return calls, (s["out"], s["keys"], s["values"]), (m, space, lib, capi)
    m = capi.DecayMixer(dense, back, rot, p("log_decay"), p("norm"), c["heads"], c["dim"], int(c["gated"]), s["scale"])
    need = lib.tbl_decay_workspace_bytes(C.byref(m), precision, 0, c["seqs"], c["tokens"])
    space = torch.empty(need, dtype=torch.uint8, device="cuda")
    args = (C.byref(m), precision, 0, EPS, p("proj"), p("states"), p("next"), *where, p("out"), space.data_ptr(), need)
    return [(lib.tbl_decay_forward, args)], (s["out"], s["next"]), (m, space, lib, capi)


def run_own(s):
    if "plan" not in s:
        s["plan"] = plan_of(s)
    calls, outputs, keep = s["plan"]
    stream = torch.cuda.current_stream().cuda_stream
    for call, args in calls:
        status = call(*args, stream)
        if status:
            keep[-1].check(status, call.__name__, keep[-2])
    return outputs


# ---- the plain forms -------------------------------------------------------------------------------------------------------------
def places(s):
    """Position of every row: [sequences, tokens]."""
    begin = s["positions"][s["slots"].long()].long()
    return begin[:, None] + torch.arange(s["case"]["tokens"], device="cuda")


def turned(s, x, weight, kind):
    """RMS norm of every head, times the weight, and rotation; x [sequences, tokens, heads, dim], worked out in `kind`."""
    c = s["case"]
    x, half = x.to(kind), c["rot_dim"] // 2
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(kind)
    if half == 0:
        return x
    cos, sin = (s[n][places(s)].to(kind)[:, :, None] for n in ("cos", "sin"))
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    pairs = c["interleaved"]
    a, b = (head[..., 0::2], head[..., 1::2]) if pairs else (head[..., :half], head[..., half:])
    u, v = a * cos - b * sin, b * cos + a * sin
    head = torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1)
    return torch.cat([head, rest], -1)


def split(s):
    c = s["case"]
    parts = s["proj"].view(c["seqs"], c["tokens"], -1).split(columns(c), -1)
    return [x.unflatten(-1, (-1, c["dim"])) if x.shape[-1] else None for x in parts]


def plain_rotate(s):
    q, k, _, _ = split(s)
    return turned(s, q, s["q_norm"], torch.float32).flatten(0, 1).to(s["dtype"]), turned(s, k, s["k_norm"], torch.float32).flatten(0, 1).to(s["dtype"])


def values_of(codes, scale, unit):
    """The numbers that codes and scales stand for, in fp32."""
    table = torch.tensor(CODES + tuple(-v for v in CODES), device=codes.device)
    return (table[codes.long()].unflatten(-1, (-1, 16)) * scale.float().unsqueeze(-1) * unit).flatten(-2)


def plain_cache4(s):
    c = s["case"]
    d, n, g = c["dim"], padded(c["dim"]), c["kv_heads"]
    q, k, v, gate = split(s)
    q = turned(s, q, s["q_norm"], torch.float32)
    k = turned(s, k, s["k_norm"], torch.float64).float()             # borders between codes: in 64 bits
    pad = lambda x: torch.nn.functional.pad(x, (0, n - d))
    new = [values_of(*rounded4(pad(x), u), u)[..., :d] for x, u in zip((k, v), s["units"])]
    row = s["cache"][s["slots"].long(), :, :c["context"]]            # [sequences, kv heads, tokens, bytes]
    codes = torch.stack([row[..., :n] & 15, row[..., :n] >> 4], -1).flatten(-2)
    scales = row[..., n:n + n // 8].contiguous().view(torch.float8_e4m3fn)
    old = [values_of(codes[..., i * n:(i + 1) * n], scales[..., i * n // 16:(i + 1) * n // 16], s["units"][i])[..., :d] for i in range(2)]
    at = places(s)
    for x, y in zip(old, new):
        x.scatter_(2, at[:, None, :, None].expand(-1, g, -1, d), y.transpose(1, 2))
    keys, values = old
    q = q.unflatten(2, (g, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)                       # [sequences, kv heads, group x tokens, dim]
    score = (q @ keys.transpose(-1, -2) * s["scale"]).unflatten(2, (-1, c["tokens"]))
    seen = torch.arange(c["context"], device="cuda") <= at[:, :, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    out = (weight.flatten(2, 3) @ values).unflatten(2, (-1, c["tokens"])) / weight.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)
    if gate is not None:
        out = out / (1.0 + torch.exp(-gate))
    return out.flatten(2).flatten(0, 1).to(s["dtype"]), new[0].flatten(0, 1), new[1].flatten(0, 1)


def plain_decay(s):
    c = s["case"]
    T, slots = c["tokens"], s["slots"].long()
    q, k, v, gate = split(s)
    q, k = turned(s, q, s["q_norm"], torch.float32), turned(s, k, s["k_norm"], torch.float32)
    q, k, v = (x.transpose(1, 2).float() for x in (q, k, v))         # [sequences, heads, tokens, dim]
    power = torch.exp(s["log_decay"].double()[:, None] * torch.arange(T + 1, device="cuda")).float()      # decay^n
    t = torch.arange(T, device="cuda")
    far = t[:, None] - t[None, :]
    mask = power[:, far.clamp(min=0)] * (far >= 0)
    first = s["states"][slots]                                       # [sequences, heads, value, key]
    o = (q @ k.transpose(-1, -2) * mask) @ v + q @ first.transpose(-1, -2) * power[:, 1:, None]
    o = (o * s["scale"]).transpose(1, 2)
    after = torch.zeros_like(s["states"])
    after[slots] = first * power[:, T, None, None] + (v * power[:, :T].flip(-1)[..., None]).transpose(-1, -2) @ k
    o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm"].view(c["heads"], -1)
    if gate is not None:
        o = o / (1.0 + torch.exp(-gate))
    return o.flatten(2).flatten(0, 1).to(s["dtype"]), after


def run(state):
    if own:
        return run_own(state)
    return {"rotate": plain_rotate, "cache4": plain_cache4, "decay": plain_decay}[state["case"]["op"]](state)


# ---- 64 bits ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    H, G, d, T, half, pairs = case["heads"], case["kv_heads"], case["dim"], case["tokens"], case["rot_dim"] // 2, case["interleaved"]
    wide = s["proj"].double().view(case["seqs"], T, -1)

    def heads_of(first, count, weight, sequence):
        """Heads `first` .. of a sequence's rows, normed and turned as complex numbers: [tokens, count, dim]."""
        x = wide[sequence, :, first * d:(first + count) * d].reshape(T, count, d)
        x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * weight.double()
        if half:
            at = torch.arange(T, device="cuda") + int(s["positions"][int(s["slots"][sequence])])
            turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
            even, odd = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if pairs else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., even].contiguous(), x[..., odd].contiguous()) * turn
            x[..., even], x[..., odd] = z.real, z.imag
        return x

    def four_bits(x, unit):
        """Numbers fp32 [..., dim] as the cache holds them, in 64 bits."""
        n, unit = x.shape[-1], unit.float()
        x = torch.nn.functional.pad(x, (0, -n % 16)).unflatten(-1, (-1, 16))
        scale = torch.minimum(x.abs().max(-1, keepdim=True).values / (unit * torch.full_like(unit, 6.0)), torch.full_like(unit, 448.0)).to(torch.float8_e4m3fn).float()
        y = torch.where(scale > 0, x / (scale * unit), torch.zeros_like(x)).double()
        grid = torch.tensor(CODES, dtype=torch.float64, device="cuda")
        low = (torch.bucketize(y.abs(), grid, right=True) - 1).clamp(max=6)
        down, up = grid[low], grid[low + 1]
        take = (y.abs() - down > up - y.abs()) | ((y.abs() - down == up - y.abs()) & (low % 2 == 1))
        return (torch.where(take, up, down) * y.sign() * scale.double() * unit.double()).flatten(-2)[..., :n]

    if case["op"] == "rotate":
        q = torch.cat([heads_of(0, H, s["q_norm"], i) for i in range(case["seqs"])])
        return q, torch.cat([heads_of(H, G, s["k_norm"], i) for i in range(case["seqs"])])
    gate = torch.sigmoid(wide[..., -H * d:]).reshape(case["seqs"], T, H, d) if case["gated"] else 1.0
    outs, keys, vals, after = [], [], [], torch.zeros_like(s["states"], dtype=torch.float64) if case["op"] == "decay" else None
    for i in range(case["seqs"]):
        q, k = heads_of(0, H, s["q_norm"], i), heads_of(H, G, s["k_norm"], i)
        v = wide[i, :, (H + G) * d:(H + 2 * G) * d].reshape(T, G, d)
        slot = int(s["slots"][i])
        begin = int(s["positions"][slot])
        out = torch.empty(T, H, d, dtype=torch.float64, device="cuda")
        if case["op"] == "cache4":
            k, v = four_bits(k.float(), s["units"][0]), four_bits(v.float(), s["units"][1])
            n = padded(d)
            for g in range(G):
                row = s["cache"][slot, g, :begin]
                sign = lambda code: 1.0 - 2.0 * (code >= 8).double()
                small = lambda code: torch.tensor(CODES, dtype=torch.float64, device="cuda")[(code % 8).long()] * sign(code)
                number = torch.empty(begin, 2 * n, dtype=torch.float64, device="cuda")
                number[:, 0::2], number[:, 1::2] = small(row[:, :n] % 16), small(row[:, :n] // 16)
                number *= row[:, n:n + n // 8].contiguous().view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)
                every_k = torch.cat([number[:, :d] * s["units"][0].double(), k[:, g]])
                every_v = torch.cat([number[:, n:n + d] * s["units"][1].double(), v[:, g]])
                hidden = torch.ones(T, T, device="cuda", dtype=torch.bool).triu(1)
                for h in range(g * (H // G), (g + 1) * (H // G)):
                    score = q[:, h] @ every_k.T * s["scale"]
                    score[:, begin:].masked_fill_(hidden, -math.inf)
                    out[:, h] = torch.softmax(score, -1) @ every_v
            keys.append(k)
            vals.append(v)
        else:
            t = torch.arange(T, device="cuda", dtype=torch.float64)
            rate = s["log_decay"].double()
            for h in range(H):
                state = s["states"][slot, h].double()
                mask = torch.exp(rate[h] * (t[:, None] - t[None, :]).clamp(min=0)).tril()
                o = (q[:, h] @ k[:, h].T * mask) @ v[:, h] + torch.exp(rate[h] * (t + 1))[:, None] * (q[:, h] @ state.T)
                o = o * s["scale"]
                out[:, h] = o / (o.square().sum(-1, keepdim=True) / d + EPS).sqrt() * s["norm"].double()[h * d:(h + 1) * d]
                after[slot, h] = torch.exp(rate[h] * T) * state + v[:, h].T @ (torch.exp(rate[h] * (T - 1 - t))[:, None] * k[:, h])
        outs.append(out * (gate[i] if case["gated"] else 1.0))
    out = torch.cat(outs).flatten(1)
    return (out, torch.cat(keys), torch.cat(vals)) if case["op"] == "cache4" else (out, after)
