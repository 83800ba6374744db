"""Packed-batch operators (rope_table, qk_norm_rope, gemm_adapters, attention_packed) against their definitions in
64 bits.

Tolerances are elementwise bounds from the roundings each kernel makes.  A value rounded to a type is off by at most
half a step, HALF[type] relative; f32 sums of n terms t_i in any order by at most n 2^-24 sum|t_i|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
HALF = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}


@pytest.fixture(scope="module")
def ctx():
    import ltx_b200
    return ltx_b200.Context(0)


def gen(*key):
    return torch.Generator(device="cuda").manual_seed(hash(tuple(int(k) for k in key)) % (1 << 31))


def normal(g, *shape, std=1.0, dtype=BF16):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def within(got, want, tol):
    """Every value of got within tol of want (both finite everywhere)."""
    got = got.to(F64)
    assert bool(torch.isfinite(got).all())
    off = (got - want).abs() - tol
    assert float(off.max()) <= 0, f"worst {float((got - want).abs().max()):.3e}, over its bound by {float(off.max()):.3e}"


# ── rope_table ───────────────────────────────────────────────────────────────

def table64(pos, rot, theta, factor, original, lo, hi, amplitude):
    f = theta ** (-2 * torch.arange(rot // 2, dtype=F64) / rot)
    w = ((original * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1) if original else torch.zeros_like(f)
    a = pos.cpu().to(F64)[:, None] * (f * w + f / factor * (1 - w))
    return a.cos().cuda() * amplitude, a.sin().cuda() * amplitude


@pytest.mark.parametrize("rows,rot,far,theta,factor,original,amplitude", [
    (1, 2, 1, 1e4, 1.0, 0, 1.0), (7, 10, 100, 1e4, 4.0, 0, 1.0), (333, 64, 1 << 20, 1e4, 16.0, 8192, 1.25),
    (1000, 128, 1 << 24, 5e5, 8.0, 4096, 0.5), (65, 510, 4096, 1e6, 1.0, 0, 1.0), (129, 80, 1 << 31, 1e4, 1.0, 0, 1.0)])
def test_rope_table(ctx, rows, rot, far, theta, factor, original, amplitude):
    import ltx_b200
    g = gen(rows, rot, far)
    pos = torch.randint(-far, far, (rows,), device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
    cos, sin = torch.full((rows, rot // 2), 9.0, device="cuda"), torch.full((rows, rot // 2), 9.0, device="cuda")
    ltx_b200.rope_table(ctx, pos, cos, sin, theta, factor, original, 1.0, 32.0, amplitude)
    ctx.synchronize()
    c, s = table64(pos, rot, theta, factor, original, 1.0, 32.0, amplitude)
    # the fraction's rounding to f32 (pi 2^-25), cos/sin to 2 ulp, the amplitude's product and the store; far positions
    # carry the f64 frequency's few 2^-53 into the angle on both sides
    tol = amplitude * (math.pi * 2.0 ** -25 + 2 * 2.0 ** -23 + 2 * 2.0 ** -24) + pos.to(F64).abs()[:, None] * 2.0 ** -49
    within(cos, c, tol)
    within(sin, s, tol)


def test_rope_table_counts_rows_without_positions(ctx):
    import ltx_b200
    cos, sin = torch.empty(50, 8, device="cuda"), torch.empty(50, 8, device="cuda")
    ltx_b200.rope_table(ctx, None, cos, sin)
    c, s = table64(torch.arange(50), 16, 1e4, 1.0, 0, 1, 32, 1.0)
    ctx.synchronize()
    within(cos, c, 5e-7)
    within(sin, s, 5e-7)


# ── qk_norm_rope ─────────────────────────────────────────────────────────────

def norm_rope64(x, heads, d, gamma, cos, sin, pos, norm, eps, interleaved):
    """(result, bound without the final rounding): x [rows, heads*d]."""
    y = x.to(F64).reshape(-1, heads, d)
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if gamma is not None:
            y = y * gamma.to(F64)
    size = y.abs()
    if cos is not None:
        rot = 2 * cos.shape[1]
        p = (torch.arange(y.shape[0], device="cuda") % cos.shape[0]) if pos is None else pos.long()
        c, s = cos.to(F64)[p][:, None], sin.to(F64)[p][:, None]
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        u, v = y[..., a].clone(), y[..., b].clone()
        y[..., a], y[..., b] = c * u - s * v, s * u + c * v
        size[..., a] = size[..., b] = u.abs() * (c.abs() + s.abs()) + v.abs() * (c.abs() + s.abs())
    # f32: the mean of d squares (d 2^-24 relative, halved by the root), a root, a division, gamma, a rotation
    return y.reshape(x.shape), (size * (d / 2 + 10) * 2.0 ** -24).reshape(x.shape)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,heads,kv,d,rot,layout,norm,gamma,pad", [
    (1, 1, 1, 128, 128, 0, True, True, 0), (5, 32, 8, 128, 128, 0, True, True, 0), (77, 4, 4, 64, 32, 1, True, True, 8),
    (130, 3, 1, 96, 96, 0, True, False, 0), (33, 2, 1, 256, 64, 1, False, False, 16), (9, 2, 2, 80, 20, 0, True, True, 0),
    (21, 3, 2, 50, 14, 1, True, True, 3), (4, 1, 0, 128, 64, 0, True, True, 0), (6, 2, 1, 1, 0, 0, True, True, 1),
    (3, 1, 1, 512, 512, 0, True, True, 0), (1025, 16, 2, 128, 0, 0, True, True, 0), (260, 9, 3, 24, 16, 0, True, True, 0)])
def test_qk_norm_rope(ctx, dtype, rows, heads, kv, d, rot, layout, norm, gamma, pad):
    import ltx_b200
    g = gen(rows, heads, d, rot, layout)
    buf = normal(g, rows, (heads + 2 * kv) * d + pad, dtype=dtype)
    q, k = buf[:, :heads * d], buf[:, heads * d:(heads + kv) * d]
    qo, ko = torch.full((rows, heads * d + pad), 7.0, device="cuda", dtype=dtype)[:, :heads * d], None
    kfull = torch.full((rows, kv * d + 2 * pad), 7.0, device="cuda", dtype=dtype)
    ko = kfull[:, pad:pad + kv * d]
    gq = 1 + normal(g, d, std=0.2, dtype=F32) if gamma else None
    gk = 1 + normal(g, d, std=0.2, dtype=F32) if gamma else None
    cos = sin = pos = None
    if rot:
        ang = torch.rand(40, rot // 2, device="cuda", generator=g) * 6.3
        cos, sin = ang.cos() * 1.1, ang.sin() * 1.1
        pos = torch.randint(0, 40, (rows,), device="cuda", generator=g, dtype=torch.int32) if rows % 2 else None
    ltx_b200.qk_norm_rope(ctx, q, k if kv else None, qo, ko if kv else None, heads, kv, cos, sin, pos=pos, gamma_q=gq,
                          gamma_k=gk, norm=norm, eps=1e-6, layout=layout)
    ctx.synchronize()
    for x, y, n, gm in ((q, qo, heads, gq), (k, ko, kv, gk)):
        if n:
            want, tol = norm_rope64(x, n, d, gm, cos, sin, pos, norm, 1e-6, layout == 1)
            # f16: values under its smallest normal have a fixed half step of 2^-25
            within(y, want, tol * (1 + HALF[dtype]) + want.abs() * HALF[dtype] + (2.0 ** -25 if dtype == F16 else 0))
    assert bool((kfull[:, :pad] == 7).all()) and bool((kfull[:, pad + kv * d:] == 7).all())


def test_qk_norm_rope_in_place_and_zero_rows(ctx):
    import ltx_b200
    g = gen(3)
    q, k = normal(g, 50, 512), normal(g, 50, 256)
    q[7] = 0
    ang = torch.rand(50, 64, device="cuda", generator=g)
    want = [norm_rope64(x, n, 128, None, ang.cos(), ang.sin(), None, True, 1e-6, False) for x, n in ((q, 4), (k, 2))]
    ltx_b200.qk_norm_rope(ctx, q, k, q, k, 4, 2, ang.cos(), ang.sin())
    ctx.synchronize()
    for x, (w, t) in zip((q, k), want):
        within(x, w, t * 1.01 + w.abs() * HALF[BF16])
    assert bool((q[7] == 0).all())
    ltx_b200.qk_norm_rope(ctx, q[:0], k[:0], q[:0], k[:0], 4, 2, ang.cos(), ang.sin())


def test_qk_norm_rope_reports_a_position_outside_the_table(ctx):
    import ltx_b200
    q = torch.ones(3, 64, device="cuda", dtype=BF16)
    t = torch.ones(4, 32, device="cuda")
    ltx_b200.qk_norm_rope(ctx, q, None, q, None, 1, 0, t, t, pos=ints([1, 4, -2]))
    with pytest.raises(ltx_b200.LtxError) as e:
        ctx.synchronize()
    assert e.value.kind == "INVALID_ARG" and "position" in str(e.value)
    ctx.synchronize()


# ── gemm_adapters ────────────────────────────────────────────────────────────

def gelu64(y):
    return y / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def adapters64(x, w, idx, a, b, coeff, epi, bias, gate, gate_idx, old):
    """(result, bound)."""
    k, rank = x.shape[1], a.shape[1]
    x, w, a, b, coeff = (t.to(F64) for t in (x, w, a, b, coeff))
    y, sums = x @ w.t(), x.abs() @ w.abs().t()
    tol = (k + rank + 4) * 2.0 ** -24 * sums
    part = HALF[BF16] ** 2 if epi in (2, 3) else HALF[BF16]      # the low-rank product in one or two bf16 parts
    for i in range(a.shape[0]):
        r = (idx == i).nonzero().flatten()
        low = coeff[i] * (x[r] @ a[i].t())
        y[r] += low @ b[i].t()
        size = coeff[i].abs() * (x[r].abs() @ a[i].abs().t())
        tol[r] += (low.abs() @ b[i].abs().t()) * (part + (k + rank + 4) * 2.0 ** -24)
        tol[r] += (size @ b[i].abs().t()) * (k + 2) * 2.0 ** -24
    if bias is not None:
        y = y + bias.to(F64)
    tol = tol + y.abs() * 2.0 ** -23
    if epi == 1:
        y, tol = gelu64(y), tol * 1.13 + gelu64(y).abs() * 2.0 ** -21 + y.abs() * 2.0 ** -22   # |gelu'| <= 1.13
    if epi == 3:
        f = gate.to(F64)[gate_idx.long() if gate_idx is not None else torch.zeros(len(y), dtype=torch.long, device="cuda")] if gate is not None else 1.0
        y, tol = old.to(F64) + y * f, tol * (f.abs() if gate is not None else 1.0) + (old.to(F64).abs() + (y * f).abs()) * 2.0 ** -23
    return y, tol + (y.abs() * HALF[BF16] if epi in (0, 1) else y.abs() * HALF[F32])


def adapter_case(ctx, m, n, k, rank, idx, epi, adapters, bias=True, gate=2, x_pad=0, o_pad=0, seed=0):
    import ltx_b200
    g = gen(m, n, k, rank, epi, seed)
    x = normal(g, m, k + x_pad)[:, :k]
    w, a = normal(g, n, k, std=0.05), normal(g, adapters, rank, k, std=0.05)
    b = normal(g, adapters, n, rank, std=0.2)
    coeff = torch.rand(adapters, device="cuda", generator=g) + 0.5
    bs = normal(g, n, dtype=F32) if bias else None
    idx = ints(idx)
    full = normal(g, m, n + o_pad, dtype=F32 if epi in (2, 3) else BF16)
    before = full.clone()
    out = full[:, :n]
    gt = normal(g, gate, n, dtype=F32) if epi == 3 and gate else None
    gi = torch.randint(0, gate, (m,), device="cuda", generator=g, dtype=torch.int32) if gt is not None and gate > 1 else None
    ltx_b200.gemm_adapters(ctx, x, w, out, idx, a, b, coeff, epilogue=epi, bias=bs, gate=gt, gate_idx=gi)
    ctx.synchronize()
    y, tol = adapters64(x, w, idx, a, b, coeff, epi, bs, gt, gi, before[:, :n])
    within(out, y, tol)
    assert torch.equal(full[:, n:], before[:, n:])


def runs(m, lengths, adapters, start=0):
    idx, i = [], start
    while len(idx) < m:
        idx += [i % (adapters + 1) - 1] * lengths[i % len(lengths)]
        i += 1
    return idx[:m]


@pytest.mark.parametrize("epi", [0, 1, 2, 3])
@pytest.mark.parametrize("m,n,k,rank,adapters,lengths", [
    (1, 8, 8, 8, 1, [1]), (1, 300, 520, 16, 3, [1]), (5, 128, 64, 8, 8, [1]), (16, 256, 512, 64, 16, [1]),
    (17, 136, 200, 24, 2, [3, 5]), (33, 1000, 256, 32, 5, [7]), (64, 64, 128, 128, 64, [1]), (100, 260, 320, 16, 4, [33, 1]),
    (130, 129, 192, 64, 3, [64, 3]), (256, 512, 512, 32, 4, [100]), (300, 384, 448, 256, 3, [77, 130]),
    (700, 640, 256, 40, 12, [1, 2, 300])])
def test_gemm_adapters(ctx, m, n, k, rank, adapters, lengths, epi):
    adapter_case(ctx, m, n, k, rank, runs(m, lengths, adapters, start=1), epi, adapters, bias=m % 3 != 0,
                 gate=(0, 1, 2)[m % 3])


@pytest.mark.parametrize("epi", [0, 1, 2, 3])
@pytest.mark.parametrize("m,n,k,rank,adapters,lengths", [
    (2100, 2601, 192, 40, 5, [300, 1, 70]), (1025, 4480, 64, 8, 3, [1024]), (513, 6500, 200, 256, 2, [400]),
    (5000, 1100, 320, 64, 40, [1])])
def test_gemm_adapters_many_tokens(ctx, m, n, k, rank, adapters, lengths, epi):
    """Enough tiles for two SMs to share one each, the last of them ragged both ways."""
    adapter_case(ctx, m, n, k, rank, runs(m, lengths, adapters, start=1), epi, adapters, bias=m % 2 == 0, gate=2)


@pytest.mark.parametrize("epi", [1, 3])
@pytest.mark.parametrize("m,n,k,rank,adapters,lengths", [
    (100, 16000, 64, 16, 2, [60]), (129, 16000, 136, 72, 3, [40, 1]), (250, 4500, 512, 32, 4, [1, 90]),
    (300, 5120, 1024, 64, 3, [128]), (400, 8300, 256, 16, 20, [1, 2, 3]), (90, 4200, 2048, 128, 5, [20])])
def test_gemm_adapters_every_tile_width(ctx, m, n, k, rank, adapters, lengths, epi):
    """Sizes for which tiles of 64 to 256 tokens are taken, alone and shared by a cluster."""
    adapter_case(ctx, m, n, k, rank, runs(m, lengths, adapters, start=1), epi, adapters, bias=True, gate=1)


@pytest.mark.parametrize("epi", [0, 3])
@pytest.mark.parametrize("m,n,k,rank,adapters,lengths", [
    (2500, 4096, 64, 72, 9, [1, 2]), (2100, 2601, 64, 200, 30, [5]), (256, 9000, 2048, 8, 2, [1]),
    (500, 2100, 128, 136, 12, [3, 1]), (64, 1000, 64, 24, 60, [1])])
def test_gemm_adapters_more_adapter_blocks_than_others(ctx, m, n, k, rank, adapters, lengths, epi):
    """Mixed tiles whose adapters take as many blocks as K or more, in ranks that fill no whole block."""
    adapter_case(ctx, m, n, k, rank, runs(m, lengths, adapters, start=1), epi, adapters, bias=False, gate=2)


def test_gemm_adapters_long_low_rank_products(ctx):
    """So many rows, each with one of 64 adapters of the largest rank, that the low-rank product alone takes a good part
    of the time that a kernel's waits may last."""
    import ltx_b200
    m, n, k, rank, adapters = (1 << 17) + 77, 72, 16384, 256, 64
    g = gen(m, k)
    x = torch.empty(m, k, device="cuda", dtype=BF16)
    for i in range(0, m, 4096):
        x[i:i + 4096] = normal(g, min(4096, m - i), k)
    w, a, b = normal(g, n, k, std=0.05), normal(g, adapters, rank, k, std=0.05), normal(g, adapters, n, rank, std=0.2)
    coeff = torch.rand(adapters, device="cuda", generator=g) + 0.5
    idx = (torch.arange(m, device="cuda") * 37 % (adapters + 1) - 1).to(torch.int32)
    out = torch.zeros(m, n, device="cuda")
    ltx_b200.gemm_adapters(ctx, x, w, out, idx, a, b, coeff, epilogue=2)
    ctx.synchronize()
    for rows in (slice(0, 300), slice(m // 2, m // 2 + 300), slice(m - 300, m)):
        y, tol = adapters64(x[rows], w, idx[rows], a, b, coeff, 2, None, None, None, None)
        within(out[rows], y, tol)


@pytest.mark.parametrize("m,n", [(20, 300), (300, 700), (2500, 4096)])
def test_gemm_adapters_after_a_call_that_left_nan(ctx, m, n):
    """What an earlier call left in the workspace, NaN here, reaches no row of a later one."""
    import ltx_b200
    x = torch.full((m, 128), float("nan"), device="cuda", dtype=BF16)
    w, a, b = (torch.ones(*s, device="cuda", dtype=BF16) for s in ((n, 128), (2, 256, 128), (2, n, 256)))
    out = torch.zeros(m, n, device="cuda")
    ltx_b200.gemm_adapters(ctx, x, w, out, ints([i % 2 for i in range(m)]), a, b, torch.ones(2, device="cuda"), epilogue=2)
    ctx.synchronize()
    assert bool(out.isnan().all())
    adapter_case(ctx, m, n, 128, 24, runs(m, [2, 1], 3), 2, 3)


@pytest.mark.parametrize("epi", [0, 3])
def test_gemm_adapters_strides_and_odd_rows(ctx, epi):
    adapter_case(ctx, 45, 77, 96, 16, runs(45, [4, 9], 3), epi, 3, x_pad=8, o_pad=3)
    adapter_case(ctx, 300, 200, 128, 16, runs(300, [4, 90], 3), epi, 3, x_pad=24, o_pad=4)


def test_one_row_of_a_matrix_of_unaligned_rows(ctx):
    """A single aligned row whose matrix has a leading dimension that 16-byte loads could not take."""
    import ltx_b200
    g = gen(62)
    buf, w = normal(g, 4, 68), normal(g, 24, 64)
    none = torch.zeros(0, 8, 64, device="cuda", dtype=BF16), torch.zeros(0, 24, 8, device="cuda", dtype=BF16)
    out = torch.zeros(1, 24, device="cuda")
    x = buf[2:3, :64]
    ltx_b200.gemm_adapters(ctx, x, w, out, ints([-1]), *none, torch.zeros(0, device="cuda"), epilogue=2)
    qkv = normal(g, 4, 3 * 64 + 4)[2:3]
    q, k, v = qkv[:, :64], qkv[:, 64:128], qkv[:, 128:192]
    o = torch.zeros(1, 64, device="cuda", dtype=BF16)
    ltx_b200.attention_packed(ctx, q, k, v, o, ints([0, 1]), ints([0, 1]), 1, 1, 1.0, head_dim=64)
    ctx.synchronize()
    within(out, x.to(F64) @ w.to(F64).t(), x.to(F64).abs() @ w.to(F64).abs().t() * 68 * 2.0 ** -24)
    assert torch.equal(o, v)


def test_one_column_of_a_larger_matrix(ctx):
    """One output, or one head of one value, that is a column of a larger matrix, its inner stride not 1."""
    import ltx_b200
    g = gen(61)
    x, w = normal(g, 5, 64), normal(g, 1, 64)
    full = torch.full((5, 6), 7.0, device="cuda")
    out = full[:, ::3][:, 1:]
    assert out.stride() == (6, 3)
    none = torch.zeros(0, 8, 64, device="cuda", dtype=BF16), torch.zeros(0, 1, 8, device="cuda", dtype=BF16)
    ltx_b200.gemm_adapters(ctx, x, w, out, ints([-1] * 5), *none, torch.zeros(0, device="cuda"), epilogue=2)
    q = torch.full((5, 6), 4.0, device="cuda")
    ltx_b200.qk_norm_rope(ctx, q[:, ::3][:, 1:], None, q[:, ::3][:, 1:], None, 1, 0, None, None, eps=0.0)
    ctx.synchronize()
    want, size = x.to(F64) @ w.to(F64).t(), x.to(F64).abs() @ w.to(F64).abs().t()
    within(out, want, size * 68 * 2.0 ** -24)
    within(q[:, 3:4], torch.ones_like(q[:, 3:4], dtype=F64), 8 * 2.0 ** -24)
    full[:, 3], q[:, 3] = 7, 4
    assert bool((full == 7).all()) and bool((q == 4).all())


@pytest.mark.parametrize("epi", [0, 2])
def test_gemm_adapters_without_any(ctx, epi):
    """Every row without an adapter is the plain projection; an empty pool too."""
    adapter_case(ctx, 70, 200, 128, 16, [-1] * 70, epi, 2)
    adapter_case(ctx, 3, 200, 128, 16, [-5, -1, -1], epi, 2)


def test_gemm_adapters_many_of_them_out_of_order(ctx):
    g = torch.Generator().manual_seed(3)
    idx = torch.randint(-1, 300, (200,), generator=g).tolist()
    adapter_case(ctx, 200, 264, 256, 16, idx, 0, 300)
    adapter_case(ctx, 200, 264, 256, 16, idx, 2, 300)


def test_gemm_adapters_empty_and_index_beyond_the_pool(ctx):
    import ltx_b200
    x, w = torch.ones(2, 64, device="cuda", dtype=BF16), torch.ones(8, 64, device="cuda", dtype=BF16)
    a, b = torch.ones(1, 8, 64, device="cuda", dtype=BF16), torch.ones(1, 8, 8, device="cuda", dtype=BF16)
    out, c = torch.zeros(2, 8, device="cuda"), torch.ones(1, device="cuda")
    ltx_b200.gemm_adapters(ctx, x[:0], w, out[:0], ints([]), a, b, c, epilogue=2)
    ltx_b200.gemm_adapters(ctx, x, w, out, ints([0, 1]), a, b, c, epilogue=2)
    with pytest.raises(ltx_b200.LtxError) as e:
        ctx.synchronize()
    assert e.value.kind == "INVALID_ARG" and "adapter" in str(e.value)
    assert out[0].tolist() == [64.0 + 64 * 8] * 8 and out[1].tolist() == [64.0] * 8
    empty = a[:0], b[:0], c[:0]
    ltx_b200.gemm_adapters(ctx, x, w, out, ints([5, 7]), *empty, epilogue=2)   # no adapters: the indices are not looked at
    ctx.synchronize()
    out.zero_()
    ltx_b200.gemm_adapters(ctx, x, w, out, ints([-1, -1]), *empty, epilogue=2)
    ctx.synchronize()
    assert bool((out == 64).all())


@pytest.mark.parametrize("m,n", [(3, 8), (300, 130), (2500, 4096)])
def test_gemm_adapters_gate_rows_outside_the_gate(ctx, m, n):
    """A gate index outside the gate takes its nearest row and is reported; every access stays inside."""
    import ltx_b200
    x, w = torch.ones(m, 64, device="cuda", dtype=BF16), torch.ones(n, 64, device="cuda", dtype=BF16)
    a, b = torch.ones(1, 8, 64, device="cuda", dtype=BF16), torch.ones(1, n, 8, device="cuda", dtype=BF16)
    rows = torch.arange(1, 4, device="cuda", dtype=F32)[:, None].expand(3, n).contiguous()
    out, c = torch.zeros(m, n, device="cuda"), torch.ones(1, device="cuda")
    idx = torch.tensor([-7, 1, 1 << 30, 2, -(1 << 31), 3], dtype=torch.int32, device="cuda").repeat(m // 6 + 1)[:m].contiguous()
    ltx_b200.gemm_adapters(ctx, x, w, out, ints([-1] * m), a, b, c, epilogue=3, gate=rows, gate_idx=idx)
    with pytest.raises(ltx_b200.LtxError) as e:
        ctx.synchronize()
    assert e.value.kind == "INVALID_ARG" and "gate" in str(e.value)
    assert torch.equal(out, 64 * rows[idx.clamp(0, 2).long()])
    out.zero_()
    ltx_b200.gemm_adapters(ctx, x, w, out, ints([-1] * m), a, b, c, epilogue=3, gate=rows, gate_idx=idx.clamp(0, 2))
    ctx.synchronize()
    assert torch.equal(out, 64 * rows[idx.clamp(0, 2).long()])


# ── attention_packed ─────────────────────────────────────────────────────────

def attention64(q, k, v, lq, lk, h, hk, d, scale, cap, slopes, causal, prefix, q0=0, k0=0):
    """(out rows of the documents, bound): per document and head in 64 bits, on the documents' own slices."""
    vt = v.dtype
    want, tol = [], []
    for i, (a, b) in enumerate(zip(lq, lk)):
        Q = q[q0:q0 + a].to(F64).reshape(a, h, d).transpose(0, 1)
        K = k[k0:k0 + b].to(F64).reshape(b, hk, d).transpose(0, 1).repeat_interleave(h // hk, 0)
        V = v[k0:k0 + b].to(F64).reshape(b, hk, d).transpose(0, 1).repeat_interleave(h // hk, 0)
        q0, k0 = q0 + a, k0 + b
        s = Q @ K.transpose(1, 2) * scale
        noise = (Q.abs() @ K.abs().transpose(1, 2) * scale).amax(-1, keepdim=True) * (d + 4) * 2.0 ** -24 if b else 0
        if cap:
            s = cap * torch.tanh(s / cap)
            noise = noise + cap * 2.0 ** -21
        place = torch.arange(a, device="cuda")[:, None] + b - a
        j = torch.arange(b, device="cuda")[None]
        if slopes is not None:
            far = slopes.to(F64)[:, None, None] * (place - j).abs()
            s = s - far
            noise = noise + (far.amax(-1, keepdim=True) * 2.0 ** -22 if b else 0)
        if causal:
            see = j <= place
            if prefix is not None:
                see = see | (j < int(prefix[i]))
            s = s.masked_fill(~see, -math.inf)
        m = s.amax(-1, keepdim=True) if b else torch.full((h, a, 1), -math.inf, device="cuda", dtype=F64)
        p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
        l = p.sum(-1, keepdim=True)
        ok = l > 0
        l = torch.where(ok, l, torch.ones_like(l))
        o = torch.where(ok, p @ V / l, torch.zeros_like(p @ V))
        mass = p @ V.abs() / l
        big = s.masked_fill(s == -math.inf, 0).abs().amax(-1, keepdim=True) if b else 0
        # P's rounding to V's type and the exponential's polynomial (1e-4) act on sum p|v|; an error e of a score changes
        # p by e; scores in the log2 domain carry their magnitude's 2^-23; f16 P under 2^-14 has a fixed step of 2^-25;
        # then f32 sums over the keys and the output's rounding
        t = mass * (HALF[vt] + 1e-4 + 2 * noise + 4 * big * 2.0 ** -23 + (b + 8) * 2.0 ** -24)
        if vt == F16:
            t = t + 2.0 ** -25 * V.abs().sum(1, keepdim=True) / l
        t = t + (o.abs() + t) * HALF[BF16]
        want.append(o.transpose(0, 1).reshape(a, h * d))
        tol.append(t.transpose(0, 1).reshape(a, h * d))
    return torch.cat(want), torch.cat(tol)


def offsets(lens, start=0):
    o = [start]
    for n in lens:
        o.append(o[-1] + n)
    return ints(o)


def attention_case(ctx, lq, lk, h, hk, d, vt=BF16, cap=0.0, slope=False, causal=False, prefix=None, spare=4, q_std=1.0,
                   start=2, poison=True, seed=0):
    import ltx_b200
    g = gen(sum(lq), sum(lk), h, d, seed)
    nq, nk = start + sum(lq) + spare, start + sum(lk) + spare
    buf = normal(g, max(nq, 1), h * d + 8, std=q_std)
    q = buf[:nq, 8:]
    kbuf = normal(g, nk, 2 * hk * d)
    k, v = kbuf[:, :hk * d], kbuf[:, hk * d:]
    if vt == F16:
        v = v.to(F16)
    if poison:     # nothing outside the documents reaches a row
        for t in (k, v):
            t[:start] = float("nan")
            t[start + sum(lk):] = float("inf")
        q[:start] = float("nan")
        q[start + sum(lq):] = float("nan")
    full = torch.full((nq, h * d + 16), 3.0, device="cuda", dtype=BF16)
    out = full[:, 8:8 + h * d]
    slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if slope else None
    pf = ints(prefix) if prefix is not None else None
    scale = 1 / math.sqrt(d)
    ltx_b200.attention_packed(ctx, q, k, v, out, offsets(lq, start), offsets(lk, start), h, hk, scale, head_dim=d,
                              softcap=cap, slopes=slopes, causal=causal, prefix=pf)
    ctx.synchronize()
    want, tol = attention64(q, k, v, lq, lk, h, hk, d, scale, cap, slopes, causal, prefix, start, start)
    within(out[start:start + sum(lq)], want, tol)
    full[start:start + sum(lq), 8:8 + h * d] = 3
    assert bool((full == 3).all())


SHAPES = [  # lq, lk, heads, kv_heads
    ([1], [1], 1, 1), ([1], [129], 2, 2), ([3, 1], [5, 77], 4, 2), ([128], [128], 2, 1), ([129], [127], 3, 3),
    ([256, 0, 40], [300, 5, 0], 4, 4), ([0, 0, 7], [0, 3, 900], 6, 2), ([257, 300], [257, 300], 5, 1),
    ([64, 1, 200], [640, 500, 13], 8, 2), ([50], [1000], 12, 4), ([33, 10], [400, 129], 16, 1)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("vt", [BF16, F16])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_packed(ctx, shape, d, vt):
    attention_case(ctx, *SHAPES[shape], d, vt)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_packed_causal(ctx, shape, d):
    """Documents with more queries than keys have rows that see nothing: they give 0."""
    attention_case(ctx, *SHAPES[shape], d, F16 if shape % 2 else BF16, causal=True)


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_packed_prefix(ctx, shape):
    lq, lk, h, hk = SHAPES[shape]
    attention_case(ctx, lq, lk, h, hk, 128, causal=True, prefix=[[0, 7, 1 << 30, 130][(i + shape) % 4] for i in range(len(lq))])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap,slope,causal", [(30.0, False, False), (0.0, True, False), (20.0, True, True), (0.0, True, True)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_packed_cap_and_distance(ctx, shape, cap, slope, causal, d):
    attention_case(ctx, *SHAPES[shape], d, F16 if shape % 2 else BF16, cap=cap, slope=slope, causal=causal,
                   q_std=4.0 if cap else 1.0)


@pytest.mark.parametrize("lq,lk,h,hk,d,kw", [
    ([1] * 5, [3000, 1, 129, 5000, 700], 8, 2, 128, dict(causal=True)),
    ([1], [20000], 2, 2, 64, {}), ([2, 1, 4], [4097, 100, 9000], 4, 4, 128, dict(causal=True, slope=True)),
    ([1] * 70, [17 * i for i in range(70)], 4, 4, 64, {}), ([5], [6000], 24, 1, 128, dict(cap=15.0, q_std=3.0)),
    ([1] * 3, [5000] * 3, 128, 1, 128, dict(causal=True)), ([3], [2500], 96, 2, 64, dict(slope=True))])
@pytest.mark.parametrize("vt", [BF16, F16])
def test_attention_packed_few_rows_long_keys(ctx, lq, lk, h, hk, d, kw, vt):
    attention_case(ctx, lq, lk, h, hk, d, vt, **kw)


@pytest.mark.parametrize("d,cap,slope", [(64, 0.0, False), (128, 0.0, True), (128, 20.0, False)])
def test_attention_packed_queries_far_ahead_of_their_keys(ctx, d, cap, slope):
    """Many more tiles than SMs, most of which see no key: a CTA takes several of them behind one that sees some."""
    attention_case(ctx, [4096], [520], 32, 32, d, causal=True, cap=cap, slope=slope)
    attention_case(ctx, [2000, 700, 1], [300, 1, 300], 16, 4, d, causal=True, prefix=[0, 1, 2], cap=cap, slope=slope)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [130, 300])
def test_attention_packed_runs_of_documents_without_keys(ctx, rows, d):
    """Runs of documents without keys behind documents of several K/V tiles, of one query tile and of two."""
    attention_case(ctx, [rows] * 400, [700 if i % 40 == 0 else 0 for i in range(400)], 2, 2, d)
    attention_case(ctx, [rows] * 400, [700 if i % 40 < 3 else 0 for i in range(400)], 2, 1, d, F16)


@pytest.mark.parametrize("causal", [False, True])
def test_attention_packed_many_short_documents(ctx, causal):
    """More documents than CTAs and than one search sees at once, some without rows or keys."""
    attention_case(ctx, [(7 * i) % 61 for i in range(900)], [(11 * i) % 83 for i in range(900)], 4, 2, 64, causal=causal)


@pytest.mark.parametrize("causal,cap,slope", [(False, 0.0, False), (True, 0.0, True), (True, 25.0, False)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_packed_rows_of_one_document_among_empty_ones(ctx, d, causal, cap, slope):
    """Few rows a document on average, nearly all of them in one: row tiles of one document behind one another on the
    line of work, documents without rows or keys between."""
    attention_case(ctx, [0, 300] + [0] * 28 + [1, 2], [700, 900] + [640, 0] * 14 + [5, 1200], 4, 2, d, causal=causal, cap=cap,
                   slope=slope)


@pytest.mark.parametrize("vt", [BF16, F16])
@pytest.mark.parametrize("cap", [0.0, 20.0, 60.0])
def test_attention_packed_few_items_share_keys(ctx, cap, vt):
    """So few items that clusters of eight share their keys, one tile each or none."""
    attention_case(ctx, [100, 30], [1100, 90], 3, 1, 128, vt, cap=cap, q_std=2.0)
    attention_case(ctx, [100, 30], [1100, 90], 2, 1, 64, vt, cap=cap, causal=True, prefix=[40, 95], q_std=2.0)


@pytest.mark.parametrize("vt", [BF16, F16])
def test_attention_packed_one_key_among_millions(ctx, vt):
    """A row that one key rules by 2^45 keeps that key's value: the sum of millions of others is nothing beside it."""
    import ltx_b200
    n, d = 1 << 23, 128
    q, k = torch.zeros(64 * 2, d, device="cuda", dtype=BF16), torch.zeros(n, d, device="cuda", dtype=BF16)
    q[:, 0], k[n // 3, 0] = 1.0, 32.0
    v = torch.ones(n, d, device="cuda", dtype=vt)
    v[n // 3] = -1.0
    out = torch.zeros(128, d, device="cuda", dtype=BF16)
    ltx_b200.attention_packed(ctx, q, k, v, out, ints([0, 128]), ints([0, n]), 1, 1, 1.0)
    ctx.synchronize()
    # the others weigh e^-32 2^23 = 1.1e-7; bf16's half step is 2e-3
    assert bool((out == -1).all())


@pytest.mark.parametrize("lq,lk", [([700, 500], [1024, 1500]), ([2], [9000])])
def test_attention_packed_row_max_grows(ctx, lq, lk):
    """Scores whose maxima grow along the keys, for some rows of a tile much faster than for others."""
    import ltx_b200
    h, d = 2, 128
    g = gen(sum(lq))
    nq, nk = sum(lq), sum(lk)
    q = normal(g, nq, h * d, dtype=F32) * (1 + 10 * (torch.rand(nq, 1, device="cuda", generator=g) > 0.5).float())
    k = normal(g, nk, h * d, dtype=F32) * (0.2 + 3 * torch.arange(nk, device="cuda")[:, None] / nk)
    q, k, v = q.to(BF16), k.to(BF16), normal(g, nk, h * d, dtype=F16)
    out = torch.zeros_like(q)
    ltx_b200.attention_packed(ctx, q, k, v, out, offsets(lq), offsets(lk), h, h, 1 / math.sqrt(d))
    ctx.synchronize()
    want, tol = attention64(q, k, v, lq, lk, h, h, d, 1 / math.sqrt(d), 0.0, None, False, None)
    within(out, want, tol)


def test_attention_packed_keeps_other_documents_values_out(ctx):
    """A document's rows are the same bits whatever its neighbours hold."""
    import ltx_b200
    g = gen(8)
    h, d, lens = 2, 128, [70, 200, 90]
    q, k, v = (normal(g, 360, h * d) for _ in range(3))
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    o = offsets(lens)
    ltx_b200.attention_packed(ctx, q, k, v, a, o, o, h, h, 0.1)
    k2, v2 = k.clone(), v.clone()
    for t in (k2, v2):
        t[:70], t[270:] = float("nan"), float("inf")
    ltx_b200.attention_packed(ctx, q, k2, v2, b, o, o, h, h, 0.1)
    ctx.synchronize()
    assert torch.equal(a[70:270], b[70:270]) and bool(torch.isfinite(a).all())


@pytest.mark.parametrize("vt,cap,causal", [(BF16, 20.0, False), (BF16, 20.0, True), (F16, 20.0, False), (BF16, 60.0, True)])
@pytest.mark.parametrize("h,hk,d", [(2, 2, 128), (3, 1, 64)])
def test_attention_packed_capped_bits_are_the_documents_own(ctx, h, hk, d, vt, cap, causal):
    """Capped scores, which have forms of tanh for small, middle and large ones: a document's rows are the same bits
    whatever its neighbours' queries, keys and values hold and whatever ran before."""
    import ltx_b200
    g = gen(h, d, int(cap))
    lens, own, n = [70, 200, 90], slice(70, 270), 360
    q, k, v = normal(g, n, h * d), normal(g, n, hk * d), normal(g, n, hk * d, dtype=vt)
    o = offsets(lens)

    def attend(q, k, v):
        out = torch.zeros(n, h * d, device="cuda", dtype=BF16)
        ltx_b200.attention_packed(ctx, q, k, v, out, o, o, h, hk, 0.2, head_dim=d, softcap=cap, causal=causal)
        return out[own]

    want = attend(q, k, v)
    for size in (30.0, 1e4, float("nan")):
        q2, k2, v2 = q * size, k * size, v * size
        attend(q2, k2, v2)          # what it leaves in shared memory
        for t, t2 in ((q, q2), (k, k2), (v, v2)):
            t2[own] = t[own]
        assert torch.equal(attend(q2, k2, v2), want)


def far_rows(q, k, v, lq, lk, rows, slope, scale):
    """Rows `rows` of one document and head in 64 bits, and a bound: the distance counts for a key's weight, from the
    nearest key on, not for the row as a whole."""
    Q, K, V = q[rows].to(F64), k[:lk].to(F64), v[:lk].to(F64)
    raw, j = Q @ K.t() * scale, torch.arange(lk, device="cuda")
    away = slope * (rows[:, None] + lk - lq - j[None]).abs().to(F64)
    p = torch.softmax(raw - away, -1)
    # a score's error: its product's sums, and the 2^-23 of its own size in the log2 domain, four roundings
    e = (Q.abs() @ K.abs().t() * scale).amax(-1, keepdim=True) * 68 * 2.0 ** -24 + \
        4 * (raw.abs() + away - away.amin(-1, keepdim=True)) * 2.0 ** -23
    o, mass = p @ V, p @ V.abs()
    # P's rounding and the exponential's polynomial as in attention64; an error of a score moves its weight and the sum
    t = mass * (HALF[BF16] + 1e-4 + (lk + 8) * 2.0 ** -24 + 2 * (p * e).sum(-1, keepdim=True)) + 2 * (p * e) @ V.abs()
    return o, t + (o.abs() + t) * HALF[BF16]


@pytest.mark.parametrize("lk,others", [(64, 0), (200, 0), (64, 16000)])
def test_attention_packed_distance_of_rows_far_from_all_keys(ctx, lk, others):
    """A million queries over a few keys: the first stand 2^20 keys before the nearest, and the weights of the keys among
    each other are those of the distances between them all the same.  Once in the kernel for few rows, which takes the
    batch where its other documents hold the most keys."""
    import ltx_b200
    lq, slope, scale = 1 << 20, 2.0 ** -0.25, 0.125
    g = gen(lk, others)
    nk = lk + 600 * others
    q, k, v = normal(g, lq + 1, 64), torch.zeros(nk, 64, device="cuda", dtype=BF16), torch.zeros(nk, 64, device="cuda", dtype=BF16)
    k[:lk], v[:lk] = normal(g, lk, 64), normal(g, lk, 64)
    out = torch.zeros_like(q)
    qo, ko = ([0, lq], [0, lk]) if not others else ([0, lq] + [lq + 1] * others, [0, lk] + [nk] * others)
    ltx_b200.attention_packed(ctx, q, k, v, out, ints(qo), ints(ko), 1, 1, scale, head_dim=64,
                              slopes=torch.tensor([slope], device="cuda"))
    ctx.synchronize()
    rows = torch.cat([torch.arange(0, 300), torch.arange(lq // 2, lq // 2 + 100), torch.arange(lq - 300, lq)]).cuda()
    want, tol = far_rows(q, k, v, lq, lk, rows, slope, scale)
    within(out[rows], want, tol)


@pytest.mark.parametrize("cap", [300.0, 3e3, 1e5, 1e8, 1e30])
@pytest.mark.parametrize("vt", [BF16, F16])
@pytest.mark.parametrize("lq,lk", [([300], [333]), ([2, 1], [3000, 777])])
def test_attention_packed_cap_far_above_the_scores(ctx, lq, lk, vt, cap):
    """A cap far above the scores hardly changes them, whatever f32 makes of 1 beside scores over the cap."""
    import ltx_b200
    h, d = 2, 128
    g = gen(sum(lq), int(math.log2(cap)))
    q, k, v = normal(g, sum(lq), h * d, std=3.0), normal(g, sum(lk), h * d), normal(g, sum(lk), h * d, dtype=vt)
    out = torch.zeros_like(q)
    ltx_b200.attention_packed(ctx, q, k, v, out, offsets(lq), offsets(lk), h, h, 1 / math.sqrt(d), softcap=cap)
    ctx.synchronize()
    # attention64's bound for uncapped scores; the capped ones differ by s^3 / 3 cap^2, which is in `want`, and the tanh
    # moves them by at most 2^-17 of themselves, or with caps up to 355 by 4e-7 of the cap (in both directions of the
    # weight and its sum)
    want, _ = attention64(q, k, v, lq, lk, h, h, d, 1 / math.sqrt(d), cap, None, False, None)
    _, tol = attention64(q, k, v, lq, lk, h, h, d, 1 / math.sqrt(d), 0.0, None, False, None)
    big = max(float((q[a:b].to(F64).view(-1, h, d).transpose(0, 1) @ k[c:e].to(F64).view(-1, h, d).permute(1, 2, 0)).abs().max())
              for a, b, c, e in zip([0, lq[0]], [lq[0], sum(lq)], [0, lk[0]], [lk[0], sum(lk)]) if b > a) / math.sqrt(d)
    vmax = float(v.abs().max())
    within(out, want, tol + 2 * vmax * (big * 2.0 ** -17 + (cap * 4e-7 if cap <= 355 else 0)))


@pytest.mark.parametrize("kw", [{}, dict(slope=True), dict(softcap=60.0), dict(softcap=20.0)])
@pytest.mark.parametrize("lq,lk", [(256, 256), (130, 512), (1, 3000)])
def test_attention_packed_a_nan_that_a_row_sees_stays_one(ctx, lq, lk, kw):
    """A NaN key makes the rows that see it NaN, wherever it stands, and no other row; a NaN query its own row."""
    import ltx_b200
    g = gen(lq, lk)
    q, k, v = normal(g, lq, 128), normal(g, lk, 128), normal(g, lk, 128).abs()
    kw = dict(kw)
    slopes = torch.full((1,), 0.01, device="cuda") if kw.pop("slope", False) else None
    place = torch.arange(lq, device="cuda") + lk - lq
    for j in (0, 1, 3, 8, 40, 64, 120, 127, 128, 201, lk - 1):
        k2 = k.clone()
        k2[j] = float("nan")
        out = torch.zeros(lq, 128, device="cuda", dtype=BF16)
        ltx_b200.attention_packed(ctx, q, k2, v, out, ints([0, lq]), ints([0, lk]), 1, 1, 0.09, causal=True, slopes=slopes, **kw)
        ctx.synchronize()
        assert torch.equal(out.isnan(), (place >= j)[:, None].expand_as(out)), j
        assert bool(out.isfinite()[place < j].all())
    q[lq // 2] = float("nan")
    out = torch.zeros(lq, 128, device="cuda", dtype=BF16)
    ltx_b200.attention_packed(ctx, q, k, v, out, ints([0, lq]), ints([0, lk]), 1, 1, 0.09, slopes=slopes, **kw)
    ctx.synchronize()
    assert torch.equal(out.isnan().all(1), torch.arange(lq, device="cuda") == lq // 2)


def test_attention_packed_the_most_documents(ctx):
    """2^24 documents, all but the last without rows: found in time; one more is refused."""
    import ltx_b200
    docs, g = 1 << 24, gen(24)
    q, k, v = normal(g, 300, 128), normal(g, 400, 128), normal(g, 400, 128)
    out = torch.zeros_like(q)
    o = torch.zeros(2, docs + 2, device="cuda", dtype=torch.int32)
    o[0, docs:], o[1, docs:] = 300, 400
    ltx_b200.attention_packed(ctx, q, k, v, out, o[0, :docs + 1], o[1, :docs + 1], 1, 1, 0.1)
    ctx.synchronize()
    want, tol = attention64(q, k, v, [300], [400], 1, 1, 128, 0.1, 0.0, None, False, None)
    within(out, want, tol)
    refused(ctx, "UNSUPPORTED", ltx_b200.attention_packed, q, k, v, out, o[0], o[1], 1, 1, 0.1)


def test_attention_packed_nothing_to_do(ctx):
    import ltx_b200
    q = torch.ones(4, 128, device="cuda", dtype=BF16)
    out = torch.full_like(q, 5.0)
    none = q[:0]
    ltx_b200.attention_packed(ctx, none, q, q, none, ints([0, 0]), ints([0, 4]), 1, 1, 1.0)
    ltx_b200.attention_packed(ctx, q, q, q, out, ints([0]), ints([0]), 1, 1, 1.0)
    ctx.synchronize()
    assert bool((out == 5).all())
    ltx_b200.attention_packed(ctx, q, none, none, out, ints([0, 3]), ints([0, 0]), 1, 1, 1.0)
    ctx.synchronize()
    assert bool((out[:3] == 0).all()) and bool((out[3] == 5).all())


def test_attention_packed_reports_bad_offsets(ctx):
    """Offsets that leave the buffers are cut to them and reported; the context stays usable."""
    import ltx_b200
    q = torch.ones(4, 128, device="cuda", dtype=BF16)
    for qo, ko in (([0, 9], [0, 4]), ([0, 4], [0, 1 << 30]), ([-7, 4], [0, 4]), ([0, 4], [3, 1])):
        out = torch.zeros_like(q)
        ltx_b200.attention_packed(ctx, q, q, q, out, ints(qo), ints(ko), 1, 1, 1.0)
        with pytest.raises(ltx_b200.LtxError) as e:
            ctx.synchronize()
        assert e.value.kind == "INVALID_ARG" and "offsets" in str(e.value)
    ctx.synchronize()


def test_a_bad_index_does_not_hide_a_wait_that_gave_up():
    """Whichever comes first, a wait that gave up is what the next synchronisation reports."""
    import ltx_b200
    ctx = ltx_b200.Context(0)
    q, t = torch.ones(3, 64, device="cuda", dtype=BF16), torch.ones(4, 32, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")

    def bad_calls():
        ltx_b200.qk_norm_rope(ctx, q, None, q, None, 1, 0, t, t, pos=ints([1, 4, -2]))
        ltx_b200.attention_packed(ctx, q, q, q, torch.zeros_like(q), ints([0, 9]), ints([0, 3]), 1, 1, 1.0, head_dim=64)
        x, w = torch.ones(2, 64, device="cuda", dtype=BF16), torch.ones(8, 64, device="cuda", dtype=BF16)
        a, b = torch.ones(1, 8, 64, device="cuda", dtype=BF16), torch.ones(1, 8, 8, device="cuda", dtype=BF16)
        out, gate = torch.zeros(2, 8, device="cuda"), torch.ones(1, 8, device="cuda")
        ltx_b200.gemm_adapters(ctx, x, w, out, ints([0, 1]), a, b, torch.ones(1, device="cuda"), epilogue=3, gate=gate,
                               gate_idx=ints([0, 1]))

    for first in (True, False):
        if not first:
            bad_calls()
        ctx.wait_flag(flag, 1, timeout_ms=20)
        if first:
            bad_calls()
        with pytest.raises(ltx_b200.LtxError) as e:
            ctx.synchronize()
        assert e.value.kind == "TIMEOUT"
    ctx.synchronize()
    bad_calls()
    with pytest.raises(ltx_b200.LtxError) as e:
        ctx.synchronize()
    assert e.value.kind == "INVALID_ARG"
    ctx.close()


# ── together, on other streams, captured ─────────────────────────────────────

def layer(ctx, s):
    """One attention layer over a packed batch, every request with its own adapter."""
    import ltx_b200 as L
    h, hk, d = s["heads"], s["kv_heads"], s["d"]
    L.gemm_adapters(ctx, s["x"], s["w_qkv"], s["qkv"], s["idx"], s["a1"], s["b1"], s["coeff"], bias=s["bias"])
    q, k, v = s["qkv"][:, :h * d], s["qkv"][:, h * d:(h + hk) * d], s["qkv"][:, (h + hk) * d:]
    L.rope_table(ctx, s["pos"], s["cos"], s["sin"], factor=4.0, original_len=512)
    L.qk_norm_rope(ctx, q, k, q, k, h, hk, s["cos"], s["sin"], gamma_q=s["gq"], gamma_k=s["gk"])
    L.attention_packed(ctx, q, k, v, s["o"], s["off"], s["off"], h, hk, 1 / math.sqrt(d), head_dim=d, causal=True,
                       prefix=s["prefix"])
    L.gemm_adapters(ctx, s["o"], s["w_o"], s["resid"], s["idx"], s["a2"], s["b2"], s["coeff"], epilogue=L.EPI_RESID,
                    gate=s["gate"])


def layer_state(seed, lens, h=4, hk=2, d=64, rank=16):
    g = gen(seed)
    n, dim = sum(lens), h * d
    idx = [i % 3 - 1 for i, m in enumerate(lens) for _ in range(m)]
    return dict(heads=h, kv_heads=hk, d=d, lens=lens, x=normal(g, n, dim), w_qkv=normal(g, (h + 2 * hk) * d, dim, std=0.06),
                qkv=torch.zeros(n, (h + 2 * hk) * d, device="cuda", dtype=BF16), idx=ints(idx),
                a1=normal(g, 2, rank, dim, std=0.06), b1=normal(g, 2, (h + 2 * hk) * d, rank, std=0.3),
                a2=normal(g, 2, rank, dim, std=0.06), b2=normal(g, 2, dim, rank, std=0.3),
                coeff=torch.tensor([0.7, 1.3], device="cuda"), bias=normal(g, (h + 2 * hk) * d, dtype=F32),
                pos=ints([j for m in lens for j in range(m)]), cos=torch.zeros(n, d // 2, device="cuda"),
                sin=torch.zeros(n, d // 2, device="cuda"), gq=1 + normal(g, d, std=0.1, dtype=F32),
                gk=1 + normal(g, d, std=0.1, dtype=F32), off=offsets(lens), prefix=ints([5] * len(lens)),
                o=torch.zeros(n, dim, device="cuda", dtype=BF16), w_o=normal(g, dim, dim, std=0.06),
                resid=normal(g, n, dim, dtype=F32), gate=normal(g, 1, dim, dtype=F32))


def layer64(s):
    h, hk, d, lens = s["heads"], s["kv_heads"], s["d"], s["lens"]
    qkv, _ = adapters64(s["x"], s["w_qkv"], s["idx"], s["a1"], s["b1"], s["coeff"], 0, s["bias"], None, None, None)
    c, sn = table64(s["pos"], d, 1e4, 4.0, 512, 1.0, 32.0, 1.0)
    q, _ = norm_rope64(qkv[:, :h * d], h, d, s["gq"], c, sn, None, True, 1e-6, False)
    k, _ = norm_rope64(qkv[:, h * d:(h + hk) * d], hk, d, s["gk"], c, sn, None, True, 1e-6, False)
    o = []
    at = 0
    for n in lens:
        Q, K, V = (t[at:at + n].reshape(n, t.shape[1] // d, d).transpose(0, 1) for t in (q, k, qkv[:, (h + hk) * d:]))
        K, V = K.repeat_interleave(h // hk, 0), V.repeat_interleave(h // hk, 0)
        i = torch.arange(n, device="cuda")
        hide = (i[None] > i[:, None]) & (i[None] >= 5)
        p = torch.softmax((Q @ K.transpose(1, 2) / math.sqrt(d)).masked_fill(hide, -math.inf), -1)
        o.append((p @ V).transpose(0, 1).reshape(n, h * d))
        at += n
    y, _ = adapters64(torch.cat(o), s["w_o"], s["idx"], s["a2"], s["b2"], s["coeff"], 3, None, s["gate"], None, s["resid"])
    return y


def rel(a, b):
    return float((a.to(F64) - b).norm() / b.norm())


# The layer's update passes four roundings to bf16 (the projection, the rotated q and k, the probabilities, the
# attention's output), each at most 2^-8 relative and independent of the others: under 2^-6 of the result's norm.
LAYER_TOL = 2.0 ** -6


@pytest.mark.parametrize("lens", [[1], [130, 1, 75], [300, 0, 257, 40]])
def test_layer_over_a_packed_batch(ctx, lens):
    s = layer_state(sum(lens), lens)
    want = layer64(s) - s["resid"].to(F64)
    before = s["resid"].to(F64)
    layer(ctx, s)
    ctx.synchronize()
    assert rel(s["resid"].to(F64) - before, want) < LAYER_TOL


def test_layer_on_its_own_stream_and_two_at_once():
    """Two contexts on streams of their own run at the same time; each result is the one it gives alone."""
    import ltx_b200
    states = [layer_state(i, lens) for i, lens in enumerate([[200, 333], [90, 7, 512]])]
    keep = [s["resid"].clone() for s in states]
    streams = [torch.cuda.Stream() for _ in states]
    ctxs = [ltx_b200.Context(0, st.cuda_stream) for st in streams]
    torch.cuda.synchronize()
    alone = []
    for c, s, k in zip(ctxs, states, keep):
        layer(c, s)
        c.synchronize()
        alone.append(s["resid"].clone())
        s["resid"].copy_(k)
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, k, st in zip(ctxs, states, keep, streams):
            with torch.cuda.stream(st):
                s["resid"].copy_(k)
            layer(c, s)
    for c in ctxs:
        c.synchronize()
    for s, a in zip(states, alone):
        assert torch.equal(s["resid"], a)
    for c in ctxs:
        c.close()


def test_layer_captured_twice_and_replayed():
    """Two graphs of one context, of different sizes, with an eager call of a third size between their replays: each
    replay gives what an eager call gives on the inputs then in its buffers."""
    import ltx_b200
    st = torch.cuda.Stream()
    ctx = ltx_b200.Context(0, st.cuda_stream)
    sizes = [[60, 70], [300, 5, 128], [700, 41]]
    a, b, c = (layer_state(10 + i, lens) for i, lens in enumerate(sizes))
    graphs = []
    torch.cuda.synchronize()
    for s in (a, b):
        layer(ctx, s)          # before the capture: the functions are loaded
        ctx.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
            layer(ctx, s)
        graphs.append(g)
    for round_ in range(3):
        for g, s in zip(graphs, (a, b)):
            fresh = layer_state(100 + round_, s["lens"])
            with torch.cuda.stream(st):
                for name in ("x", "resid", "idx"):
                    s[name].copy_(fresh[name])
                keep = s["resid"].clone()
                g.replay()
                got = s["resid"].clone()
                s["resid"].copy_(keep)
            layer(ctx, c)
            layer(ctx, s)
            ctx.synchronize()
            assert torch.equal(s["resid"], got)
    del graphs
    ctx.close()


def test_first_calls_of_a_context_captured():
    """A context whose very first calls are captured, in the strictest capture mode: workspaces and pools come into being
    under the capture."""
    import ltx_b200
    st = torch.cuda.Stream()
    ctx = ltx_b200.Context(0, st.cuda_stream)
    s = layer_state(31, [90, 3])
    keep = s["resid"].clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        layer(ctx, s)
    with torch.cuda.stream(st):
        g.replay()
        got = s["resid"].clone()
        s["resid"].copy_(keep)
    layer(ctx, s)
    ctx.synchronize()
    assert torch.equal(s["resid"], got) and not torch.equal(got, keep)
    del g
    ctx.close()


def test_large_workspaces_go_back_to_the_device():
    """What one call needs beyond 64 MB is free for other allocators after the next synchronisation."""
    import ltx_b200
    ctx = ltx_b200.Context(0)
    m, rank = 1 << 18, 256          # 2 parts x m x rank x 2 bytes: 256 MB
    x, w = torch.ones(m, 8, device="cuda", dtype=BF16), torch.ones(8, 8, device="cuda", dtype=BF16)
    a, b = torch.ones(1, rank, 8, device="cuda", dtype=BF16), torch.ones(1, 8, rank, device="cuda", dtype=BF16)
    c, out, idx = torch.ones(1, device="cuda"), torch.zeros(m, 8, device="cuda"), torch.zeros(m, device="cuda", dtype=torch.int32)
    ltx_b200.gemm_adapters(ctx, x[:256], w, out[:256], idx[:256], a, b, c, epilogue=2)
    ctx.synchronize()
    before = torch.cuda.mem_get_info(0)[0]
    for _ in range(2):
        ltx_b200.gemm_adapters(ctx, x, w, out, idx, a, b, c, epilogue=2)
        ctx.synchronize()
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info(0)[0] <= 96 << 20
    assert bool((out == 8 + 8 * rank).all())
    ctx.close()


# ── refusals of the C entry points ───────────────────────────────────────────

def refused(ctx, kind, fn, *args, **kw):
    import ltx_b200
    with pytest.raises(ltx_b200.LtxError) as e:
        fn(ctx, *args, **kw)
    assert e.value.kind == kind, str(e.value)


def test_refusals(ctx):
    import ltx_b200 as L
    t = torch.zeros(4, 32, device="cuda")
    refused(ctx, "SHAPE", L.rope_table, None, torch.zeros(4, 300, device="cuda"), torch.zeros(4, 300, device="cuda"))
    refused(ctx, "INVALID_ARG", L.rope_table, None, t, t, theta=-1.0)
    refused(ctx, "INVALID_ARG", L.rope_table, None, t, t, factor=0.0)
    refused(ctx, "INVALID_ARG", L.rope_table, None, t, t, original_len=8, turns_low=2.0, turns_high=2.0)
    q = torch.zeros(4, 128, device="cuda", dtype=BF16)
    refused(ctx, "SHAPE", L.qk_norm_rope, q, None, q, None, 4, 0, t, t)              # 64 rotated of heads of 32
    refused(ctx, "INVALID_ARG", L.qk_norm_rope, q, None, q, None, 1, 0, t[:0], t[:0])
    refused(ctx, "INVALID_ARG", L.qk_norm_rope, q, None, q, None, 1, 0, t, t, layout=2)
    refused(ctx, "INVALID_ARG", L.qk_norm_rope, q, None, q, None, 1, 0, t, t, eps=-1.0)
    o = ints([0, 4])
    ok = (q, q, q, torch.zeros_like(q), o, o)
    refused(ctx, "UNSUPPORTED", L.attention_packed, *ok, 4, 4, 1.0, head_dim=32)
    refused(ctx, "INVALID_ARG", L.attention_packed, *ok, 1, 1, 0.0)
    refused(ctx, "INVALID_ARG", L.attention_packed, *ok, 1, 1, float("nan"))
    refused(ctx, "INVALID_ARG", L.attention_packed, *ok, 1, 1, 1.0, softcap=-1.0)
    refused(ctx, "INVALID_ARG", L.attention_packed, *ok, 1, 1, 1.0, prefix=ints([1]))
    refused(ctx, "INVALID_ARG", L.attention_packed, *ok, 1, 1, 3e38)
    refused(ctx, "INVALID_ARG", L.attention_packed, *ok, 1, 1, 1.0, softcap=1e-39)
    three = torch.zeros(4, 384, device="cuda", dtype=BF16)
    two = torch.zeros(4, 256, device="cuda", dtype=BF16)
    refused(ctx, "SHAPE", L.attention_packed, three, two, two, three, o, o, 3, 2, 1.0)
    odd = torch.zeros(4, 133, device="cuda", dtype=BF16)
    refused(ctx, "SHAPE", L.attention_packed, odd[:, 1:129], q, q, q, o, o, 1, 1, 1.0)
    x, w, i = torch.zeros(4, 64, device="cuda", dtype=BF16), torch.zeros(8, 64, device="cuda", dtype=BF16), ints([0] * 4)
    c, y = torch.ones(1, device="cuda"), torch.zeros(4, 8, device="cuda", dtype=BF16)

    def pool(r, k=64):
        return torch.zeros(1, r, k, device="cuda", dtype=BF16), torch.zeros(1, 8, r, device="cuda", dtype=BF16), c

    refused(ctx, "UNSUPPORTED", L.gemm_adapters, x, w, y, i, *pool(12))
    refused(ctx, "UNSUPPORTED", L.gemm_adapters, x, w, y, i, *pool(264))
    refused(ctx, "INVALID_ARG", L.gemm_adapters, x, w, y, i, *pool(8), epilogue=7)
    refused(ctx, "SHAPE", L.gemm_adapters, x[:, :60], w[:, :60], y, i, *pool(8, 60))
    gate = torch.zeros(1, 8, device="cuda")
    refused(ctx, "SHAPE", L.gemm_adapters, x, w, torch.zeros(4, 8, device="cuda"), i, *pool(8), epilogue=3, gate=gate[:0])
    refused(ctx, "INVALID_ARG", L.rope_table, None, t, t, amplitude=1e39)
    refused(ctx, "DTYPE", L.gemm_adapters, x, w, y, i, *pool(8), epilogue=3, gate=gate)
    ctx.synchronize()
