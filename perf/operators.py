"""What is measured of the packed-batch operators: a batch of requests whose rows lie one behind another in one
buffer, each request with its own length and its own low-rank adapter.  One attention layer over such a batch runs
gemm_adapters (the projection with every request's adapter beside the shared weight), rope_table and qk_norm_rope
(each head's norm and the rotation by position in one pass) and attention_packed (no request sees another's keys).

`run` computes a case with elementary torch operations where `own` is false, and with the calls of ltx_b200 where it
is true.  `exact` computes the same from the definitions in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    return [
        # the smallest attention: two short captions read by a few tokens each, where the call's latency counts
        _attention("attn_captions", docs=2, rows=41, keys=154, spare=3, heads=8, kv_heads=8, dim=64),
        # three clips of unequal length denoised as one batch: the widest self-attention of the 22B model's heads
        _attention("attn_clips", docs=3, rows=8192, keys=8192, heads=32, kv_heads=32, dim=128, v_f16=True),
        # a reference clip every token sees, then the tokens in order, scores capped
        _attention("attn_prefix_capped", docs=5, rows=4099, keys=4099, heads=16, kv_heads=4, dim=128, causal=True,
                   prefix=256, softcap=30.0),
        # one new token per request over what each has cached, keys that count less the farther they lie
        _attention("attn_one_token", docs=16, rows=16, keys=70001, heads=32, kv_heads=8, dim=128, causal=True,
                   slopes=True),
        # one row per request (a timestep's modulation, a new token), every request with an adapter of its own
        _adapters("proj_one_row_each", rows=8, n=4096, k=4096, rank=16, adapters=8, run=1, epilogue="bf16"),
        # key and value projections of a ragged batch of text contexts
        _adapters("proj_context_kv", rows=1003, n=8192, k=4096, rank=32, adapters=6, run=190, epilogue="bf16"),
        # the first feed-forward projection of two clips' tokens, GELU
        _adapters("proj_ffn_gelu", rows=4096, n=16384, k=4096, rank=128, adapters=2, run=2100, epilogue="gelu"),
        # the attention's output projection into the gated residual stream, at the full token count
        _adapters("proj_out_residual", rows=12288, n=4096, k=4096, rank=64, adapters=4, run=2600, epilogue="resid"),
        # a few new tokens' queries and keys
        _norm_rope("norm_rope_tokens", rows=16, heads=32, kv_heads=8, dim=128, rot=128, dtype="bf16", layout="half"),
        # queries and keys of a clip at the full token count, part of each head rotated
        _norm_rope("norm_rope_clip", rows=12288, heads=32, kv_heads=32, dim=128, rot=96, dtype="bf16",
                   layout="interleaved"),
        # angles of a short context
        _table("table_context", rows=1024, rot=64, far=1024, factor=1.0, original=0),
        # angles of a long context, the slow frequencies stretched past the length the model learned
        _table("table_long", rows=131072, rot=128, far=1 << 20, factor=16.0, original=8192),
    ]


def _attention(name, docs, rows, keys, heads, kv_heads, dim, spare=0, v_f16=False, causal=False, prefix=0,
               softcap=0.0, slopes=False):
    return dict(name=name, op="attention", docs=docs, rows=rows, keys=keys, heads=heads, kv_heads=kv_heads, dim=dim,
                spare=spare, v_f16=v_f16, causal=causal, prefix=prefix, softcap=softcap, slopes=slopes)


def _adapters(name, rows, n, k, rank, adapters, run, epilogue):
    return dict(name=name, op="adapters", rows=rows, n=n, k=k, rank=rank, adapters=adapters, run=run,
                epilogue=epilogue)


def _norm_rope(name, rows, heads, kv_heads, dim, rot, dtype, layout):
    return dict(name=name, op="norm_rope", rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, dtype=dtype,
                layout=layout)


def _table(name, rows, rot, far, factor, original):
    return dict(name=name, op="table", rows=rows, rot=rot, far=far, factor=factor, original=original)


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "adapters", "adapters", "norm_rope", "table"])
    if op == "attention":
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([g for g in (1, 1, 2, 3, 4, 8) if g * kv <= 32])
        docs = _log(rng, 1, 40)
        dim = rng.choice([64, 128, 128])
        if rng.random() < 0.35:   # a few new tokens per request over a long cache
            rows, keys = docs * rng.randint(1, 4), _log(rng, 200, 70000)
        elif rng.random() < 0.4:  # tokens over a context
            rows, keys = _log(rng, 32, 8192), _log(rng, 32, 2048)
        else:                     # a request's tokens among themselves
            rows = keys = _log(rng, 32, 8192)
        causal = rng.random() < 0.5
        return {k: v for k, v in _attention(
            "", docs, rows, keys, kv * group, kv, dim, spare=rng.choice([0, 0, 5]), v_f16=rng.random() < 0.5,
            causal=causal, prefix=_log(rng, 1, 600) if causal and rng.random() < 0.5 else 0,
            softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3).items() if k != "name"}
    if op == "adapters":
        rows = _log(rng, 1, 12288)
        n, k = 8 * _log(rng, 32, 768 if rows > 4096 else 2048), 64 * _log(rng, 4, 64)
        return {k_: v for k_, v in _adapters(
            "", rows, n, k, rng.choice([8, 16, 32, 64, 128]), rng.randint(1, 12), _log(rng, 1, max(1, rows)),
            rng.choice(["bf16", "gelu", "f32", "resid"])).items() if k_ != "name"}
    if op == "norm_rope":
        kv = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 96, 128, 256])
        return {k: v for k, v in _norm_rope(
            "", _log(rng, 1, 8192), kv * rng.choice([1, 2, 4]), kv, dim, dim // rng.choice([1, 1, 2, 4]),
            rng.choice(["bf16", "f16", "f32"]), rng.choice(["half", "interleaved"])).items() if k != "name"}
    return {k: v for k, v in _table("", _log(rng, 1, 131072), rng.choice([32, 64, 80, 128]), _log(rng, 100, 1 << 24),
                                    rng.choice([1.0, 4.0, 16.0]), rng.choice([0, 4096, 8192])).items() if k != "name"}


def _lengths(total, docs, key):
    """`docs` unequal lengths that add up to `total` (some may be 0 when total is small)."""
    r = random.Random("%d %d %s" % (total, docs, key))
    w = [r.uniform(0.25, 1.0) for _ in range(docs)]
    cuts, acc = [0], 0.0
    for x in w:
        acc += x
        cuts.append(round(total * acc / sum(w)))
    cuts[-1] = total
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _doc_lengths(case):
    if case["rows"] == case["keys"]:
        q = _lengths(case["rows"], case["docs"], "both")
        return q, q
    if case["rows"] % case["docs"] == 0:
        return [case["rows"] // case["docs"]] * case["docs"], _lengths(case["keys"], case["docs"], "keys")
    return _lengths(case["rows"], case["docs"], "rows"), _lengths(case["keys"], case["docs"], "keys")


def _limits(case, lq, lk):
    """For each query row of one request: how many of its first keys it sees."""
    if not case["causal"]:
        return [lk] * lq
    return [max(min(case["prefix"], lk), min(lk, max(0, i + lk - lq + 1))) for i in range(lq)]


def _adapter_of_row(case):
    """The adapter of each row: runs of `run` rows, now and then a run without one (-1)."""
    r = random.Random("%d %d %d" % (case["rows"], case["run"], case["adapters"]))
    idx = []
    while len(idx) < case["rows"]:
        a = -1 if r.random() < 0.1 else r.randrange(case["adapters"])
        idx += [a] * min(r.randint((case["run"] + 1) // 2, case["run"]), case["rows"] - len(idx))
    return idx


# ── inputs ───────────────────────────────────────────────────────────────────

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = {"case": case}
    if case["op"] == "attention":
        lq, lk = _doc_lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        # queries and keys come out of a norm: unit values; capped scores are large ones
        s["q"] = normal(case["rows"] + case["spare"], h * d, std=3.0 if case["softcap"] else 1.0)
        s["k"] = normal(case["keys"] + case["spare"], hk * d)
        s["v"] = normal(case["keys"] + case["spare"], hk * d, dtype=F16 if case["v_f16"] else BF16)
        s["out"] = torch.zeros_like(s["q"])
        s["q_offsets"] = ints([0] + [sum(lq[:i + 1]) for i in range(len(lq))])
        s["k_offsets"] = ints([0] + [sum(lk[:i + 1]) for i in range(len(lk))])
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["slopes"] else None
        s["prefix"] = ints([min(case["prefix"], n) for n in lk]) if case["prefix"] else None
        s["scale"] = 1.0 / math.sqrt(d)
    elif case["op"] == "adapters":
        m, n, k, r, a = (case[x] for x in ("rows", "n", "k", "rank", "adapters"))
        s["x"] = normal(m, k)
        s["w"] = normal(n, k, std=0.02)
        s["bias"] = normal(n, std=0.02, dtype=F32)
        s["a"] = normal(a, r, k, std=0.02)
        s["b"] = normal(a, n, r, std=0.02)
        s["coeff"] = torch.rand(a, device="cuda", generator=g) + 0.5
        s["idx"] = ints(_adapter_of_row(case))
        s["out"] = (normal(m, n, dtype=F32) if case["epilogue"] == "resid" else
                    torch.empty(m, n, device="cuda", dtype=F32 if case["epilogue"] == "f32" else BF16))
        s["gate"] = normal(2, n, dtype=F32) if case["epilogue"] == "resid" else None
        s["gate_idx"] = ints([int(i >= m // 2) for i in range(m)]) if case["epilogue"] == "resid" else None
    elif case["op"] == "norm_rope":
        t = {"bf16": BF16, "f16": F16, "f32": F32}[case["dtype"]]
        h, hk, d, m = case["heads"], case["kv_heads"], case["dim"], case["rows"]
        s["qkv"] = normal(m, (h + 2 * hk) * d, dtype=t)   # the fused projection's output
        s["q"], s["k"] = s["qkv"][:, :h * d], s["qkv"][:, h * d:(h + hk) * d]
        s["q_out"], s["k_out"] = torch.empty(m, h * d, device="cuda", dtype=t), torch.empty(m, hk * d, device="cuda", dtype=t)
        s["gq"], s["gk"] = 1 + normal(d, std=0.1, dtype=F32), 1 + normal(d, std=0.1, dtype=F32)
        ang = torch.rand(4096, case["rot"] // 2, device="cuda", generator=g) * 6.28
        s["cos"], s["sin"] = ang.cos(), ang.sin()
        s["pos"] = torch.randint(0, 4096, (m,), device="cuda", generator=g, dtype=torch.int32)
    else:
        m = case["rows"]
        s["pos"] = torch.randint(0, case["far"], (m,), device="cuda", generator=g, dtype=torch.int32)
        s["cos"] = torch.empty(m, case["rot"] // 2, device="cuda")
        s["sin"] = torch.empty(m, case["rot"] // 2, device="cuda")
    return s


def work(case):
    if case["op"] == "attention":
        lq, lk = _doc_lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(sum(_limits(case, a, b)) for a, b in zip(lq, lk))
        return {"bytes": 2 * d * (2 * sum(lq) * h + 2 * sum(lk) * hk), "flops": 4 * d * h * pairs}
    if case["op"] == "adapters":
        m, n, k, r = (case[x] for x in ("rows", "n", "k", "rank"))
        idx = [i for i in _adapter_of_row(case) if i >= 0]
        out = {"bf16": 2, "gelu": 2, "f32": 4, "resid": 8}[case["epilogue"]]
        return {"bytes": 2 * (m * k + n * k + len(set(idx)) * r * (n + k)) + out * m * n,
                "flops": 2 * m * n * k + 2 * len(idx) * r * (n + k)}
    if case["op"] == "norm_rope":
        e = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * e * (4 if case["dtype"] == "f32" else 2) + case["rows"] * (case["rot"] * 4 + 4), "flops": 8 * e}
    return {"bytes": case["rows"] * (4 + 4 * case["rot"]), "flops": 8 * case["rows"] * case["rot"]}


# ── one pass ─────────────────────────────────────────────────────────────────

_context = None


def _ltx():
    """The library and one context of it, as a program that uses it keeps them."""
    global _context
    if _context is None:
        if os.path.join(ROOT, "ltx-rust_b200") not in sys.path:
            sys.path.insert(0, os.path.join(ROOT, "ltx-rust_b200"))
        import ltx_b200
        _context = (ltx_b200, ltx_b200.Context(0))
    return _context


def run(s):
    return {"attention": _run_attention, "adapters": _run_adapters, "norm_rope": _run_norm_rope,
            "table": _run_table}[s["case"]["op"]](s)


def _run_attention(s):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    if own:
        ltx, ctx = _ltx()
        ltx.attention_packed(ctx, s["q"], s["k"], s["v"], s["out"], s["q_offsets"], s["k_offsets"], h, hk, s["scale"],
                             head_dim=d, softcap=c["softcap"], slopes=s["slopes"], causal=c["causal"],
                             prefix=s["prefix"])
        return s["out"]
    nq, nk, docs = s["q"].shape[0], s["k"].shape[0], c["docs"]
    qo, ko = s["q_offsets"].long(), s["k_offsets"].long()
    i, j = torch.arange(nq, device="cuda"), torch.arange(nk, device="cuda")
    doc_i, doc_j = (i[:, None] >= qo[None, 1:]).sum(1), (j[:, None] >= ko[None, 1:]).sum(1)   # docs = behind the last
    inside = doc_i < docs
    di = doc_i.clamp(max=docs - 1)
    k0, lk = ko[di], ko[di + 1] - ko[di]
    place = i - qo[di] + lk - (qo[di + 1] - qo[di])       # the key a query stands beside: requests end together
    limit = lk
    if c["causal"]:
        limit = torch.minimum(lk, (place + 1).clamp(min=0))
        if s["prefix"] is not None:
            limit = torch.maximum(limit, torch.minimum(s["prefix"].long()[di], lk))
    rel = j[None, :] - k0[:, None]
    seen = inside[:, None] & (doc_i[:, None] == doc_j[None, :]) & (rel < limit[:, None])
    q = s["q"].float().view(nq, hk, h // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
    x = torch.matmul(q, s["k"].float().view(nk, hk, d).permute(1, 2, 0)).view(h, nq, nk)
    x *= s["scale"]
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    if s["slopes"] is not None:
        x -= s["slopes"][:, None, None] * (place[:, None] - rel).abs().float()[None]
    x = torch.where(seen[None], x, torch.full((), -math.inf, device="cuda"))
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(hk, -1, nk), s["v"].float().view(nk, hk, d).permute(1, 0, 2)).view(h, nq, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(1, 0, 2).reshape(nq, h * d)
    return torch.where(inside[:, None], o.to(BF16), s["out"])


def _run_adapters(s):
    c = s["case"]
    if own:
        ltx, ctx = _ltx()
        epi = {"bf16": ltx.EPI_BF16, "gelu": ltx.EPI_GELU_BF16, "f32": ltx.EPI_F32, "resid": ltx.EPI_RESID}[c["epilogue"]]
        ltx.gemm_adapters(ctx, s["x"], s["w"], s["out"], s["idx"], s["a"], s["b"], s["coeff"], epilogue=epi,
                          bias=s["bias"], gate=s["gate"], gate_idx=s["gate_idx"])
        return s["out"]
    x, a, r = s["x"].float(), c["adapters"], c["rank"]
    y = torch.matmul(x, s["w"].float().t())
    low = torch.matmul(x, s["a"].float().view(a * r, -1).t()).view(-1, a, r)
    mine = s["idx"][:, None] == torch.arange(a, device="cuda", dtype=torch.int32)[None]
    low = low * (mine.float() * s["coeff"][None])[:, :, None]
    y = y + torch.matmul(low.view(-1, a * r), s["b"].float().permute(0, 2, 1).reshape(a * r, -1)) + s["bias"]
    if c["epilogue"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if c["epilogue"] == "resid":
        return s["out"].add_(y * s["gate"][s["gate_idx"].long()])
    return y if c["epilogue"] == "f32" else y.to(BF16)


def _run_norm_rope(s):
    c = s["case"]
    d, rot = c["dim"], c["rot"]
    if own:
        ltx, ctx = _ltx()
        ltx.qk_norm_rope(ctx, s["q"], s["k"], s["q_out"], s["k_out"], c["heads"], c["kv_heads"], s["cos"], s["sin"],
                         pos=s["pos"], gamma_q=s["gq"], gamma_k=s["gk"], eps=1e-6,
                         layout=ltx.ROPE_HALF if c["layout"] == "half" else ltx.ROPE_INTERLEAVED)
        return s["q_out"], s["k_out"]
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]

    def one(x, heads, gamma):
        y = x.float().reshape(-1, heads, d)
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * gamma
        if c["layout"] == "half":
            u, v, rest = y[..., :rot // 2], y[..., rot // 2:rot], y[..., rot:]
            y = torch.cat([cos * u - sin * v, sin * u + cos * v, rest], -1)
        else:
            u, v, rest = y[..., 0:rot:2], y[..., 1:rot:2], y[..., rot:]
            y = torch.cat([torch.stack([cos * u - sin * v, sin * u + cos * v], -1).flatten(-2), rest], -1)
        return y.reshape(-1, heads * d).to(x.dtype)

    return one(s["q"], c["heads"], s["gq"]), one(s["k"], c["kv_heads"], s["gk"])


THETA, TURNS_LOW, TURNS_HIGH, AMPLITUDE = 10000.0, 1.0, 32.0, 1.25


def _run_table(s):
    c = s["case"]
    amplitude = AMPLITUDE if c["original"] else 1.0
    if own:
        ltx, ctx = _ltx()
        ltx.rope_table(ctx, s["pos"], s["cos"], s["sin"], theta=THETA, factor=c["factor"], original_len=c["original"],
                       turns_low=TURNS_LOW, turns_high=TURNS_HIGH, amplitude=amplitude)
        return s["cos"], s["sin"]
    # 64 bits: a far position's angle has thousands of turns before its fraction
    f = THETA ** (-2.0 * torch.arange(c["rot"] // 2, device="cuda", dtype=F64) / c["rot"])
    if c["original"]:
        keep = ((f * c["original"] / (2 * math.pi) - TURNS_LOW) / (TURNS_HIGH - TURNS_LOW)).clamp(0, 1)
        f = f * keep + f / c["factor"] * (1 - keep)
    else:
        f = f / c["factor"]
    ang = s["pos"].to(F64)[:, None] * f[None]
    return (torch.cos(ang) * amplitude).float(), (torch.sin(ang) * amplitude).float()


# ── the definitions in 64 bits ───────────────────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "adapters": _exact_adapters, "norm_rope": _exact_norm_rope,
            "table": _exact_table}[case["op"]](case, s)


def _exact_attention(c, s):
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    out = s["out"].to(F64)
    q0 = k0 = 0
    for lq, lk in zip(*_doc_lengths(c)):
        lim = torch.tensor(_limits(c, lq, lk), device="cuda", dtype=torch.long)
        at = torch.arange(lk, device="cuda")
        for e in range(h):
            kv = e // (h // hk)
            q = s["q"][q0:q0 + lq, e * d:(e + 1) * d].to(F64)
            k = s["k"][k0:k0 + lk, kv * d:(kv + 1) * d].to(F64)
            v = s["v"][k0:k0 + lk, kv * d:(kv + 1) * d].to(F64)
            t = q @ k.t() * s["scale"]
            if c["softcap"]:
                t = torch.tanh(t / c["softcap"]) * c["softcap"]
            if c["slopes"]:
                own_place = torch.arange(lq, device="cuda") + (lk - lq)
                t = t - float(s["slopes"][e]) * (own_place[:, None] - at[None]).abs()
            hidden = at[None] >= lim[:, None]
            p = torch.softmax(t.masked_fill(hidden, -math.inf), -1) if lk else t
            p = p.masked_fill((lim == 0)[:, None], 0.0)
            out[q0:q0 + lq, e * d:(e + 1) * d] = p @ v
        q0, k0 = q0 + lq, k0 + lk
    return out


def _exact_adapters(c, s):
    y = s["x"].to(F64) @ s["w"].to(F64).t()
    idx = s["idx"].long()
    for a in range(c["adapters"]):
        rows = (idx == a).nonzero().flatten()
        y[rows] += float(s["coeff"][a]) * (s["x"][rows].to(F64) @ s["a"][a].to(F64).t()) @ s["b"][a].to(F64).t()
    y += s["bias"].to(F64)
    if c["epilogue"] == "gelu":
        y = y / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    if c["epilogue"] == "resid":
        y = s["out"].to(F64) + y * s["gate"].to(F64)[s["gate_idx"].long()]
    return y


def _exact_norm_rope(c, s):
    both = []
    for x, heads, gamma in ((s["q"], c["heads"], s["gq"]), (s["k"], c["kv_heads"], s["gk"])):
        x = x.to(F64).unflatten(1, (heads, c["dim"]))
        x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + 1e-6) * gamma.to(F64)
        half = c["rot"] // 2
        first = torch.arange(half, device="cuda") * (1 if c["layout"] == "half" else 2)
        second = first + (half if c["layout"] == "half" else 1)
        turn = torch.complex(s["cos"].to(F64), s["sin"].to(F64))[s["pos"].long()][:, None]
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        both.append(x.flatten(1))
    return tuple(both)


def _exact_table(c, s):
    i = torch.arange(c["rot"] // 2, device="cuda", dtype=F64)
    f = torch.exp(-math.log(THETA) * i * 2 / c["rot"])
    amplitude = 1.0
    if c["original"]:
        turns = c["original"] * f / (2 * math.pi)
        w = torch.clamp((turns - TURNS_LOW) / (TURNS_HIGH - TURNS_LOW), 0, 1)
        f, amplitude = f * (w + (1 - w) / c["factor"]), AMPLITUDE
    else:
        f = f / c["factor"]
    a = torch.outer(s["pos"].to(F64), f)
    return a.cos() * amplitude, a.sin() * amplitude
