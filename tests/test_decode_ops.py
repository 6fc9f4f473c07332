"""The operators of a decoding step against plain implementations in fp64: RMS norm (and its 8-bit output), rotary positions and the
paged cache, attention of one new token over that cache, and log-probabilities of given tokens.

Tolerances are derived, element by element. U[t] is half a step of the output type relative to the value; E = 2^-24 is that of fp32,
in which all sums and statistics are held. A sum of n terms in a chain is off by at most n E times the sum of magnitudes."""
import math

import numpy as np
import pytest
import torch

from docc_b200 import _lib, ops

E = 2.0**-24
U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}  # half the smallest step near zero
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


def close(got, want, tol):
    """Every element within its tolerance; NaN and infinities have to agree."""
    got = got.detach().double().cpu()
    want, tol = want.double().cpu(), torch.as_tensor(tol, dtype=torch.float64).cpu().expand(want.shape)
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    off = (got - want).abs()[fine] - tol[fine]
    assert off.numel() == 0 or off.max() <= 0, f"off by {off.max():.3g} more than allowed"


def settle():
    ops.sync()
    torch.cuda.synchronize()


def normal(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- RMS norm ---------------------------------------------------------------------------------------------------------------------
def rms_exact(x, gamma, residual, eps):
    s = x.double() if residual is None else x.double() + residual.double()
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s, y if gamma is None else y * gamma.double()


def rms_tolerance(y, cols):
    # sum of squares: a chain of at most cols / 32 terms per lane and ten joins, halved by the root; sum, root, two products: 8 E
    return y.abs() * (cols / 32 + 10 + 8) * E


RMS_SHAPES = [(1, 1), (1, 7), (3, 64), (5, 127), (2, 128), (4, 129), (7, 257), (3, 1000), (33, 1024), (2, 4096), (3, 5003), (2, 8200),
              (2, 16384), (1, 32768), (300, 512), (1500, 256), (1300, 333), (1200, 1023)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", RMS_SHAPES)
@pytest.mark.parametrize("extra", ["plain", "gamma", "both"])
def test_rmsnorm(rt, rows, cols, dtype, extra):
    x = normal(rows, cols, seed=rows * 7 + cols, dtype=dtype)
    gamma = 1 + 0.3 * normal(cols, seed=5) if extra != "plain" else None
    residual = 2 * normal(rows, cols, seed=9, dtype=dtype) if extra == "both" else None
    s, y = rms_exact(x, gamma, residual, 1e-5)
    got = ops.rmsnorm(x.cuda(), None if gamma is None else gamma.cuda(), None if residual is None else residual.cuda(), eps=1e-5)
    settle()
    if residual is not None:
        got, total = got
        close(total, s, s.abs() * (U[dtype] + E) + TINY[dtype])
    close(got, y, y.abs() * U[dtype] * 1.01 + rms_tolerance(y, cols) + TINY[dtype])


def quantised(y, group):
    rows, cols = y.shape
    width = cols if group == 0 else 128
    scale = torch.stack([p.abs().amax(1) / 448 for p in y.split(width, dim=1)], 1)
    return scale, scale.repeat_interleave(width, dim=1)[:, :cols]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", RMS_SHAPES)
@pytest.mark.parametrize("group", [0, 128])
def test_rmsnorm_quant(rt, rows, cols, dtype, group):
    x = normal(rows, cols, seed=rows + cols, dtype=dtype)
    gamma, residual = 1 + 0.3 * normal(cols, seed=5), 2 * normal(rows, cols, seed=9, dtype=dtype)
    s, y = rms_exact(x, gamma, residual, 1e-6)
    q, scales, total = ops.rmsnorm_quant(x.cuda(), gamma.cuda(), residual.cuda(), eps=1e-6, group=group)
    settle()
    scale, wide = quantised(y, group)
    close(total, s, s.abs() * (U[dtype] + E) + TINY[dtype])
    drift = (cols / 32 + 10 + 8 + 2) * E  # of y, and of the scale with its division
    close(scales, scale, scale * drift)
    # e4m3: half a step is 2^-4 of the value and 2^-10 below the smallest normal number; a value that the drift moves over the middle
    # between two codes is off by that much more
    close(q.cpu().float().double() * scales.cpu().double().repeat_interleave(128 if group else cols, dim=1)[:, :cols], y,
          y.abs() * (2.0**-4 + 4 * drift) + wide * 2.0**-10 * (1 + 4 * drift))


@gpu
@pytest.mark.parametrize("group", [0, 128])
def test_rmsnorm_quant_zero_rows_nan_and_tiny(rt, group):
    x = normal(5, 300, seed=1)
    x[1] = 0
    x[2, 200] = float("nan")
    x[3] *= 1e-30
    x[4, 7] = float("inf")
    q, scales = ops.rmsnorm_quant(x.cuda(), group=group, eps=0.0 if group else 1e-6)
    settle()
    q, scales = q.cpu().float(), scales.cpu()
    if group == 0:
        assert (q[1] == 0).all() and scales[1] == 0
        assert torch.isnan(scales[4]).all() and torch.isnan(q[4]).all()  # inf * 0 in one place, one scale for the row
    else:
        assert torch.isnan(q[1]).all()  # 0 * rsqrt(0): as the formula has it without eps
    assert torch.isnan(scales[2]).all() and torch.isnan(q[2]).all()  # the row's mean square is NaN
    assert torch.isfinite(scales[0]).all() and q[0].abs().max() == 448


@gpu
@pytest.mark.parametrize("cols", [512, 515])
def test_rmsnorm_in_place_and_strided(rt, cols):
    wide = normal(6, 2 * cols + 8, seed=3, dtype=torch.bfloat16).cuda()
    x = wide[:, :cols]
    r = wide[:, cols : 2 * cols]
    want = ops.rmsnorm(x.contiguous(), None, r.contiguous())
    got = ops.rmsnorm(x, None, r)
    settle()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # S into the residual's own buffer, Y into the input's
    x2, r2 = x.contiguous(), r.contiguous()
    ops.call("docc_b200_rmsnorm", ord("b"), 6, cols, x2.data_ptr(), cols, r2.data_ptr(), cols, None, 1e-6, r2.data_ptr(), x2.data_ptr(), 0)
    settle()
    assert torch.equal(x2, want[0]) and torch.equal(r2, want[1])


@gpu
def test_rmsnorm_of_host_arrays_and_unaligned_views(rt):
    x, g = normal(9, 130, seed=2), 1 + normal(130, seed=3)
    s, y = rms_exact(x, g, x, 1e-6)
    got, total = ops.rmsnorm(x.numpy(), g.numpy(), x.numpy())
    close(torch.from_numpy(got), y, y.abs() * E + rms_tolerance(y, 130))
    close(torch.from_numpy(total), s, s.abs() * E)
    q, scales = ops.rmsnorm_quant(x.numpy(), g.numpy(), group=128)
    q2, scales2 = ops.rmsnorm_quant(x.cuda(), g.cuda(), group=128)
    settle()
    assert q.dtype == np.uint8 and np.array_equal(q, q2.view(torch.uint8).cpu().numpy()) and np.array_equal(scales, scales2.cpu().numpy())
    flat = normal(1 + 4 * 256, seed=4).cuda()
    view = flat[1:].view(4, 256)  # starts 4 bytes off a 16-byte boundary
    a, b = ops.rmsnorm(view), ops.rmsnorm(view.clone())
    settle()
    close(a, b, b.double().abs().cpu() * (256 / 32 + 18) * 2 * E)
    assert ops.rmsnorm(torch.empty(0, 8, device="cuda")).shape == (0, 8)


# ---- rotary positions ---------------------------------------------------------------------------------------------------------------
def rope_exact(x, positions, freq, interleaved, mscale, sign=1):
    half = len(freq)
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    angle = positions.double()[:, None] * torch.as_tensor(freq)[None]
    cos, sin = mscale * torch.cos(angle)[:, None], sign * mscale * torch.sin(angle)[:, None]
    y, x = x.double().clone(), x.double()
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    reach = x.abs().clone()
    reach[..., a] = reach[..., b] = mscale * (x[..., a].abs() + x[..., b].abs())
    return y, reach


def rope_tolerance(y, reach, dtype):
    # reduced angle: half a step of fp32 at half a turn, 2 pi 2^-25; sine and cosine: 2 steps; products and their sum: 3 E
    return y.abs() * U[dtype] * 1.01 + reach * (math.pi * 2.0**-24 + 2.0**-22 + 4 * E) + TINY[dtype]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rotary", [(1, 1, 2, 2), (1, 32, 128, 128), (7, 3, 80, 80), (5, 4, 96, 48), (33, 2, 64, 10),
                                                     (3, 5, 256, 64), (2, 1, 7, 6), (4, 2, 128, 0), (600, 8, 64, 64)])
def test_rope(rt, tokens, heads, dim, rotary, interleaved, dtype):
    x = normal(tokens, heads, dim, seed=dim + rotary, dtype=dtype)
    positions = torch.randint(0, 2_000_000, (tokens,), generator=torch.Generator().manual_seed(2))
    positions[0] = 0
    positions[-1] = 1_999_999_999
    freq, mscale = ops.rope_frequencies(rotary)
    got = ops.rope(x.cuda(), positions.cuda(), torch.from_numpy(freq).cuda(), interleaved=interleaved, mscale=1.25)
    back = ops.rope(got, positions.cuda(), torch.from_numpy(freq).cuda(), interleaved=interleaved, inverse=True)
    same = x.cuda()
    ops.rope(same, positions.cuda(), torch.from_numpy(freq).cuda(), interleaved=interleaved, mscale=1.25, out=same)
    settle()
    y, reach = rope_exact(x, positions, freq, interleaved, 1.25)
    # fp64 turns: position 2^31 times 2^-53 of a turn more
    close(got, y, rope_tolerance(y, reach, dtype) + reach * 2 * math.pi * 2.0**-21 * 2.0**-1)
    assert torch.equal(got, same)
    assert torch.equal(got[..., rotary:].cpu(), x[..., rotary:])
    y2, reach2 = rope_exact(got.cpu(), positions, freq, interleaved, 1.0, sign=-1)
    close(back, y2, rope_tolerance(y2, reach2, dtype) + reach2 * 2 * math.pi * 2.0**-22)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_inverse_is_the_gradient(rt, interleaved):
    """<g, rope(x + h) - rope(x - h)> = <inverse(g), 2 h>: the map is linear, so differences are exact up to rounding."""
    x, h, g = (normal(6, 2, 32, seed=s).cuda() for s in (1, 2, 3))
    positions, freq = torch.arange(6).cuda() * 1000, torch.from_numpy(ops.rope_frequencies(24)[0]).cuda()
    turn = lambda t, inverse=False: ops.rope(t.contiguous(), positions, freq, interleaved=interleaved, mscale=1.5, inverse=inverse)
    up, down, grad = turn(x + h), turn(x - h), turn(g, True)
    settle()
    left, right = (g.double() * (up.double() - down.double())).sum(), (grad.double() * 2 * h.double()).sum()
    room = (g.double().abs() * 4 * 1.5 * (x.abs() + h.abs()).double()).sum()  # each factor's error is a few E of its terms
    assert abs(left - right) <= room * 16 * E


@gpu
def test_rope_of_strided_views_and_host_arrays(rt):
    packed = normal(9, 3 * 4 * 24, seed=5, dtype=torch.float16).cuda()
    positions, freq = torch.arange(9), torch.from_numpy(ops.rope_frequencies(16)[0])
    view = packed[:, 96:192].unflatten(1, (4, 24))
    want = ops.rope(view.contiguous(), positions.cuda(), freq.cuda())
    got = ops.rope(view, positions.cuda(), freq.cuda())
    settle()
    assert torch.equal(got, want)
    before = packed.clone()
    ops.rope(view, positions.cuda(), freq.cuda(), out=view)
    settle()
    assert torch.equal(view, want) and torch.equal(packed[:, :96], before[:, :96]) and torch.equal(packed[:, 192:], before[:, 192:])
    host = ops.rope(view.cpu().contiguous().numpy(), positions.numpy(), freq.numpy())
    again = ops.rope(view.contiguous(), positions.cuda(), freq.cuda())
    settle()
    assert np.array_equal(host, again.cpu().numpy())


def test_rope_frequencies():
    freq, m = ops.rope_frequencies(8, base=10000.0)
    assert np.allclose(freq, [1.0, 0.1, 0.01, 0.001], rtol=1e-15) and m == 1.0
    assert np.allclose(ops.rope_frequencies(8, scaling="linear", factor=4)[0], freq / 4, rtol=1e-15)
    ntk = ops.rope_frequencies(8, scaling="ntk", factor=4)[0]
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], freq[-1] / 4, rel_tol=1e-12)
    yarn, m = ops.rope_frequencies(128, scaling="yarn", factor=8, original_length=4096)
    plain = ops.rope_frequencies(128)[0]
    turns = 4096 * plain / (2 * math.pi)
    assert np.array_equal(yarn[turns > 40], plain[turns > 40]) and np.allclose(yarn[turns < 0.8], plain[turns < 0.8] / 8, rtol=1e-15)
    assert (np.diff(yarn) < 0).all() and math.isclose(m, 0.1 * math.log(8) + 1)
    assert ops.rope_frequencies(0)[0].shape == (0,)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="yarn", factor=2), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=2, scaling="ntk", factor=2), dict(rotary_dim=8, base=1.0)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(**bad)


# ---- the cache ------------------------------------------------------------------------------------------------------------------------
def cache_pair(pages, kv, page, dim, dtype, layout, seed=0):
    """Two caches as [pages, kv, page, dim] tensors, contiguous ("hsd") or views of [pages, page, kv, dim] ("shd")."""
    shape = (pages, kv, page, dim) if layout == "hsd" else (pages, page, kv, dim)
    k, v = normal(*shape, seed=seed, dtype=dtype).cuda(), normal(*shape, seed=seed + 1, dtype=dtype).cuda()
    return (k, v) if layout == "hsd" else (k.transpose(1, 2), v.transpose(1, 2))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["hsd", "shd"])
@pytest.mark.parametrize("tokens,heads,kv,dim,rotary,page,interleaved", [(1, 4, 4, 64, 64, 16, False), (9, 8, 2, 128, 128, 16, True),
                                                                         (5, 3, 1, 80, 40, 7, False), (40, 6, 3, 7, 4, 1, True),
                                                                         (300, 4, 2, 64, 64, 24, False)])
def test_rope_append(rt, tokens, heads, kv, dim, rotary, page, interleaved, layout, dtype):
    qkv = normal(tokens, (heads + 2 * kv) * dim, seed=tokens, dtype=dtype)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, kv * dim, kv * dim], dim=1))
    dq, dk, dv = (x.unflatten(1, (-1, dim)) for x in qkv.cuda().split([heads * dim, kv * dim, kv * dim], dim=1))
    pages = tokens // page + 2
    kc, vc = cache_pair(pages, kv, page, dim, dtype, layout)
    k0, v0 = kc.cpu().clone(), vc.cpu().clone()
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:tokens]
    if tokens > 4:
        slots[2] = -1
    positions = torch.arange(tokens) + 7777
    freq = torch.from_numpy(ops.rope_frequencies(rotary)[0])
    out = ops.rope_append(dq, dk, dv, positions.cuda(), freq.cuda(), kc, vc, slots.cuda(), interleaved=interleaved, mscale=0.75)
    settle()
    y, reach = rope_exact(q, positions, freq, interleaved, 0.75)
    close(out, y, rope_tolerance(y, reach, dtype))
    yk, reach = rope_exact(k, positions, freq, interleaved, 0.75)
    written = torch.zeros(pages, page, dtype=torch.bool)
    for t in range(tokens):
        if slots[t] < 0:
            continue
        p, o = divmod(int(slots[t]), page)
        written[p, o] = True
        close(kc[p, :, o], yk[t], rope_tolerance(yk[t], reach[t], dtype))
        assert torch.equal(vc[p, :, o].cpu(), v[t])
    keep = ~written[:, None, :, None].expand(pages, kv, page, dim)
    assert torch.equal(kc.cpu()[keep], k0[keep]) and torch.equal(vc.cpu()[keep], v0[keep])


@gpu
def test_rope_append_reports_a_slot_past_the_end(rt):
    q, k, v = normal(3, 2, 64, seed=1).cuda(), normal(3, 2, 64, seed=2).cuda(), normal(3, 2, 64, seed=3).cuda()
    whole = torch.zeros(2, 5, 2, 4, 64, device="cuda")  # pages 1..3 are the cache; what lies around it must stay
    kc, vc = whole[0, 1:4], whole[1, 1:4]
    freq = torch.from_numpy(ops.rope_frequencies(64)[0]).cuda()
    slots = torch.tensor([11, 12, 2**62], device="cuda")
    settle()
    ops.rope_append(q, k, v, torch.arange(3).cuda(), freq, kc, vc, slots)
    with pytest.raises(_lib.DoccB200Error) as e:
        ops.sync()
    assert e.value.status == 7 and "slot" in str(e.value)
    ops.sync()  # reported once
    torch.cuda.synchronize()
    assert torch.equal(vc[2, :, 3], v[0]) and (whole[:, 0] == 0).all() and (whole[:, 4] == 0).all() and int((whole[1] != 0).sum()) == 128


# ---- attention over the cache -------------------------------------------------------------------------------------------------------------
def attention_exact(q, kc, vc, table, lengths, scale, softcap, window, chain=None):
    """Output and lse in fp64 with their tolerances; pages outside the cache are left out."""
    B, H, D = q.shape
    pages, kv, page, _ = kc.shape
    out, lse = torch.zeros(B, H, D, dtype=torch.float64), torch.full((B, H), -math.inf, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    kd, vd = kc.double().cpu(), vc.double().cpu()
    pv = 2.0**-16 if q.dtype != torch.float32 else 0.0  # 16-bit inputs: probabilities may enter the product as two 16-bit parts
    for b in range(B):
        n = max(0, min(int(lengths[b]), table.shape[1] * page))
        j = torch.arange(max(0, n - window) if window else 0, n)
        at = table[b].long()[j // page] if n else j
        ok = (at >= 0) & (at < pages)
        j, at = j[ok], at[ok]
        if len(j) == 0:
            continue
        for h in range(H):
            k, v = kd[at, h // (H // kv), j % page], vd[at, h // (H // kv), j % page]
            x = q[b, h].double()
            s = (k @ x) * scale
            # a score: a chain of D products, the scale; the cap adds a division, tanh (2 steps) and a product, none above |s|
            es = float((k.abs() @ x.abs()).max() * abs(scale) * (D + 4) * E)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                es += 6 * E * softcap
            m = s.max()
            # exp: the difference and its product with log2 e are rounded, |s - m| 2 E, and the function adds 4 E
            ep = 2 * es + float((m - s).clamp(max=100).max()) * 3 * E + 6 * E
            p = torch.exp(s - m)
            total = p.sum()
            p = p / total
            n_chain = (len(j) + 40) * E
            out[b, h] = p @ v
            out_tol[b, h] = (p @ v.abs()) * (2 * ep + 2 * n_chain + pv)
            lse[b, h] = m + torch.log(total)
            lse_tol[b, h] = es + ep + n_chain + lse[b, h].abs() * 2 * E
    return out, out_tol + out.abs() * U[q.dtype] * 1.01 + TINY[q.dtype], lse, lse_tol


def paged_problem(lengths, heads, kv, dim, page, dtype, layout="hsd", seed=0, spare=2):
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(need) + spare
    kc, vc = cache_pair(pages, kv, page, dim, dtype, layout, seed=seed + 10)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    table, used = torch.zeros(len(lengths), max(need + [1]), dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[used : used + n]
        table[b, n:] = order[-1]
        used += n
    q = 2 * normal(len(lengths), heads, dim, seed=seed + 3, dtype=dtype)
    return q, kc, vc, table, torch.tensor(lengths, dtype=torch.int32)


def check_paged(problem, softcap=0.0, window=0, scale=None):
    q, kc, vc, table, lengths = problem
    got, lse = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda(), scale=scale, softcap=softcap, window=window, return_lse=True)
    settle()
    out, out_tol, want_lse, lse_tol = attention_exact(q, kc, vc, table, lengths, 1 / math.sqrt(q.shape[2]) if scale is None else scale, softcap, window)
    close(got, out, out_tol)
    close(lse, want_lse, lse_tol)
    return got, lse


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (8, 2, 128), (4, 4, 80), (6, 2, 96), (16, 1, 64), (7, 1, 128), (40, 2, 64), (2, 1, 256),
                                          (3, 1, 40), (2, 2, 7), (5, 1, 130), (4, 1, 16), (2, 1, 200)])
@pytest.mark.parametrize("page,lengths", [(16, [1, 0, 17, 300, 64, 128]), (24, [129, 5, 1000]), (1, [70]), (64, [63, 64, 65, 0]), (7, [0, 0])])
def test_paged_attention(rt, heads, kv, dim, page, lengths, dtype):
    check_paged(paged_problem(lengths, heads, kv, dim, page, dtype))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["hsd", "shd"])
@pytest.mark.parametrize("softcap,window", [(0.0, 1), (0.0, 50), (5.0, 0), (30.0, 129), (0.0, 10**9)])
def test_paged_attention_cap_window_and_layout(rt, softcap, window, layout, dtype):
    check_paged(paged_problem([1, 0, 200, 51, 777], 8, 2, 64, 16, dtype, layout), softcap, window)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,heads,kv,dim", [([5000], 8, 1, 128), ([3000, 0, 1, 4500, 20, 2], 4, 2, 64), ([1] * 70, 2, 2, 64),
                                                  ([257] * 40, 8, 8, 64), ([0] * 3 + [6000], 2, 1, 256)])
def test_paged_attention_split_and_joined(rt, lengths, heads, kv, dim, dtype):
    check_paged(paged_problem(lengths, heads, kv, dim, 16, dtype))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_ignores_what_it_must_not_see(rt, dtype):
    """NaN and infinities behind the length, before the window, and on pages that no sequence owns change nothing."""
    q, kc, vc, table, lengths = paged_problem([37, 130, 0], 4, 2, 64, 16, dtype)
    clean = check_paged((q, kc, vc, table, lengths), window=20)
    seen = torch.zeros(kc.shape[0], 16, dtype=torch.bool)
    for b, n in enumerate(lengths.tolist()):
        for j in range(max(0, n - 20), n):
            seen[table[b, j // 16], j % 16] = True
    hide = ~seen[:, None, :, None].expand(kc.shape).cuda()
    kc[hide] = float("nan")
    vc[hide] = float("inf")
    settle()
    got = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda(), window=20, return_lse=True)
    settle()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_extreme_scores(rt, dtype):
    """The type's lowest value as a key element (a mask written into the cache), keys whose every score is -inf, and large scores."""
    q, kc, vc, table, lengths = paged_problem([40, 40, 40], 2, 1, 64, 16, dtype)
    q = q.abs() + 0.5
    rows = lambda b, j: (int(table[b, j // 16]), 0, j % 16)
    for j in range(30):
        kc[rows(0, j)] = torch.finfo(dtype).min / 128
    for j in range(40):
        kc[rows(1, j)] = -float("inf")
        kc[rows(2, j)] *= 30
    settle()
    got, lse = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda(), return_lse=True)
    settle()
    out, out_tol, want_lse, lse_tol = attention_exact(q[[0, 2]], kc, vc, table[[0, 2]], lengths[[0, 2]], 1 / 8, 0.0, 0)
    if dtype == torch.float16:  # finite scores: the whole row is held to the formula
        close(got[[0, 2]], out, out_tol)
        close(lse[[0, 2]], want_lse, lse_tol)
    else:  # the scores of the masked keys overflow to -inf or are far below: only the ten visible keys count
        visible = attention_exact(q[[0]], kc, vc, table[[0]], lengths[[0]], 1 / 8, 0.0, 10)
        close(got[[0]], visible[0], visible[1])
        close(got[[2]], out[[1]], out_tol[[1]])
    assert (got[1] == 0).all() and (lse[1] == -math.inf).all()


@gpu
def test_paged_attention_reports_bad_pages_and_lengths(rt):
    q, kc, vc, table, lengths = paged_problem([50, 20], 2, 1, 64, 16, torch.bfloat16)
    table[0, 1] = kc.shape[0]
    table[1, 1] = -5
    settle()
    got = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda())
    with pytest.raises(_lib.DoccB200Error) as e:
        ops.sync()
    assert e.value.status == 7 and "page" in str(e.value)
    torch.cuda.synchronize()
    out, tol, _, _ = attention_exact(q, kc, vc, table, lengths, 1 / 8, 0.0, 0)
    close(got, out, tol)
    table = table.clamp(0, kc.shape[0] - 1)
    lengths = torch.tensor([10**6, -3], dtype=torch.int32)
    got = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda())
    with pytest.raises(_lib.DoccB200Error) as e:
        ops.sync()
    assert e.value.status == 7 and "length" in str(e.value)
    ops.sync()
    torch.cuda.synchronize()
    out, tol, _, _ = attention_exact(q, kc, vc, table, lengths, 1 / 8, 0.0, 0)
    close(got, out, tol)


@gpu
def test_paged_attention_beyond_32_bit_offsets(rt):
    """A cache of more than 2^32 elements; the sequence's pages lie at its end."""
    pages = (2**32 + 2**22) // (16 * 128)
    kc = torch.zeros(pages, 1, 16, 128, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros(pages, 1, 16, 128, dtype=torch.bfloat16, device="cuda")
    q = normal(1, 2, 128, seed=1, dtype=torch.bfloat16)
    freq = torch.from_numpy(ops.rope_frequencies(128)[0]).cuda()
    n = 40
    at = torch.tensor([pages - 1, pages - 7, 3])
    slots = at[torch.arange(n) // 16] * 16 + torch.arange(n) % 16
    k, v = normal(n, 1, 128, seed=2, dtype=torch.bfloat16), normal(n, 1, 128, seed=3, dtype=torch.bfloat16)
    settle()
    ops.rope_append(k.cuda(), k.cuda(), v.cuda(), torch.zeros(n, dtype=torch.int64).cuda(), freq, kc, vc, slots.cuda())
    got = ops.paged_attention(q.cuda(), kc, vc, at[None].int().cuda(), torch.tensor([n], dtype=torch.int32).cuda())
    settle()
    small_k, small_v = kc[at.cuda()].cpu(), vc[at.cuda()].cpu()
    assert torch.equal(small_k.transpose(1, 2).reshape(-1, 128)[:n], k[:, 0]) and torch.equal(small_v.transpose(1, 2).reshape(-1, 128)[:n], v[:, 0])
    out, tol, _, _ = attention_exact(q, small_k, small_v, torch.arange(3)[None].int(), torch.tensor([n]), 1 / math.sqrt(128), 0.0, 0)
    close(got, out, tol)


# ---- log-probabilities ----------------------------------------------------------------------------------------------------------------------
def check_logprobs(x, ids, k, scale=1.0, device=None):
    logp, entropy, top_ids, top_logp = ops.token_logprobs(x.cuda() if device is None else device, ids.cuda(), k=k, scale=scale)
    settle()
    rows, vocab = x.shape
    z = x.double() * scale
    lse = torch.logsumexp(z, 1, keepdim=True)
    lp = z - lse
    m = z.amax(1)
    spread = torch.where(torch.isfinite(z), m[:, None] - z, 0).amax(1).clamp(max=110)
    # terms: argument rounded (3 E of the spread), function 4 E; the sum: a chain of at most vocab / 32 terms and 20 joins
    s0 = (3 * spread + 4 + vocab / 32 + 20) * E
    base = s0 + lse[:, 0].abs() * 2 * E + 4 * E
    keep = (ids >= 0) & (ids < vocab)
    want = torch.where(keep, lp.gather(1, ids.clamp(0, vocab - 1)[:, None])[:, 0], torch.nan)
    reach = torch.where(torch.isfinite(want), want, 0).abs() + lse[:, 0].abs()
    close(logp, want, base + 3 * E * reach)
    p = torch.exp(lp)
    h = -torch.where(p > 0, p * lp, 0).sum(1)
    log_s0 = (lse[:, 0] - m).abs()
    close(entropy, h, 2 * s0 + (log_s0 + (h - log_s0).abs()) * (2 * s0 + 4 * E) + 4 * E)
    assert top_ids.shape == (rows, k) and top_ids.dtype == torch.int64
    values, order = torch.sort(x.double(), dim=1, descending=True, stable=True)
    assert torch.equal(top_ids.cpu(), order[:, :k])
    picked = lp.gather(1, order[:, :k])
    # scale * x may leave fp32's range: a value of magnitude 2^128 or more lies half a step or further above the largest finite
    # number, so its rounding to the fp32 output is an infinity
    picked = torch.where(picked <= -(2.0**128), -math.inf, picked)
    close(top_logp, picked, base[:, None] + 3 * E * (torch.where(torch.isfinite(picked), picked, 0).abs() + lse.abs()))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (1, 1, 0), (3, 31, 31), (2, 33, 32), (5, 1000, 5), (1, 32000, 20), (4, 50021, 32), (2, 131072, 1),
                                          (150, 4096, 20), (300, 517, 3), (9, 200000, 20), (40, 10007, 0), (700, 2048, 8)])
def test_token_logprobs(rt, rows, vocab, k, dtype):
    x = 3 * normal(rows, vocab, seed=rows + vocab, dtype=dtype)
    ids = torch.randint(vocab, (rows,), generator=torch.Generator().manual_seed(4))
    check_logprobs(x, ids, k)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "steps"])
@pytest.mark.parametrize("vocab,k", [(64, 32), (5000, 32), (40000, 20)])
def test_token_logprobs_ties_and_sorted_rows(rt, vocab, k, order, dtype):
    x = {"rising": torch.linspace(-5, 5, vocab), "falling": torch.linspace(5, -5, vocab), "equal": torch.zeros(vocab),
         "steps": (torch.arange(vocab) % 7).float()}[order].expand(3, vocab).clone()
    x[1] *= -1  # -0 and 0 are equal
    x[2, vocab // 2 :] -= 1
    check_logprobs(x.to(dtype), torch.tensor([0, vocab - 1, vocab // 2]), k)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_masks_scale_and_strides(rt, dtype):
    x = 4 * normal(6, 3001, seed=8, dtype=dtype)
    x[0, 100:] = -float("inf")  # masked vocabulary
    x[1, :2990] = torch.finfo(dtype).min
    x[2, 5] = 80.0  # nearly all mass on one token
    ids = torch.tensor([3, 2995, 5, -1, 3001, 2**40])
    check_logprobs(x, ids, 12, scale=0.5)
    wide = torch.full((6, 3100), float("nan"), dtype=dtype)
    wide[:, 37:3038] = x
    check_logprobs(x, ids, 12, scale=2.0, device=wide.cuda()[:, 37:3038])


@gpu
def test_token_logprobs_nan_and_empty_distribution(rt):
    x = normal(3, 500, seed=2)
    x[0, 77] = float("nan")
    x[1] = -float("inf")
    logp, entropy, top_ids, top_logp = ops.token_logprobs(x.cuda(), torch.zeros(3, dtype=torch.int64).cuda(), k=3)
    settle()
    assert torch.isnan(logp[:2]).all() and torch.isnan(entropy[:2]).all() and torch.isnan(top_logp[:2]).all() and torch.isfinite(logp[2])
    assert top_ids[0, 0] == 77 and top_ids[1].tolist() == [0, 1, 2]


@gpu
def test_token_logprobs_of_host_arrays(rt):
    x = 3 * normal(4, 777, seed=1)
    ids = torch.tensor([0, 5, 776, 12])
    host = ops.token_logprobs(x.numpy(), ids.numpy(), k=4)
    dev = ops.token_logprobs(x.cuda(), ids.cuda(), k=4)
    settle()
    for a, b in zip(host, dev):
        assert np.array_equal(a, b.cpu().numpy())


# ---- refusals -------------------------------------------------------------------------------------------------------------------------------
def test_refusals_of_host_calls():
    f = np.zeros((2, 3, 8), dtype=np.float32)
    pos, freq, slots = np.zeros(2, dtype=np.int64), np.zeros(4), np.zeros(2, dtype=np.int64)
    cache = np.zeros((2, 3, 4, 8), dtype=np.float32)
    with pytest.raises(TypeError):
        ops.rope_append(f, f, f, pos, freq, cache, cache, slots)
    with pytest.raises(TypeError):
        ops.paged_attention(f, cache, cache, np.zeros((2, 1), dtype=np.int32), np.zeros(2, dtype=np.int32))
    with pytest.raises(TypeError):
        ops.rmsnorm(f, torch.zeros(8))
    with pytest.raises(TypeError):
        ops.rmsnorm(torch.zeros(2, 8))
    with pytest.raises(TypeError):
        ops.rmsnorm(f, np.zeros(8))  # gamma must be float32
    with pytest.raises(ValueError):
        ops.rmsnorm(f, np.zeros(7, dtype=np.float32))
    with pytest.raises(ValueError):
        ops.rmsnorm(f, residual=np.zeros((2, 8), dtype=np.float32))
    with pytest.raises(ValueError):
        ops.rmsnorm_quant(f, group=64)
    with pytest.raises(ValueError):
        ops.rmsnorm(f[:, :, ::2])
    with pytest.raises(TypeError):
        ops.rope(f, pos.astype(np.int32), freq)
    with pytest.raises(ValueError):
        ops.rope(f, pos[:1], freq)
    with pytest.raises(ValueError):
        ops.rope(f, pos, np.zeros(5))
    with pytest.raises(TypeError):
        ops.rope(f, pos, freq.astype(np.float32))
    with pytest.raises(TypeError):
        ops.token_logprobs(f[0], np.zeros(3, dtype=np.int32))
    with pytest.raises(ValueError):
        ops.token_logprobs(f, pos)


@pytest.mark.parametrize("k", [-1, 9, 33, 10**15])
def test_token_logprobs_refuses_a_k_without_allocating_for_it(k):
    with pytest.raises(_lib.DoccB200Error) as e:
        ops.token_logprobs(np.zeros((2, 8), dtype=np.float32), np.zeros(2, dtype=np.int64), k=k)
    assert e.value.status == 1


@gpu
@pytest.mark.parametrize("k", [-1, 9, 33, 10**15])
def test_token_logprobs_refuses_a_k_on_the_device(rt, k):
    with pytest.raises(_lib.DoccB200Error) as e:
        ops.token_logprobs(torch.zeros(2, 8, device="cuda"), torch.zeros(2, dtype=torch.int64).cuda(), k=k)
    assert e.value.status == 1


def status_of(name, *args):
    return getattr(_lib.lib(), name)(*args)


def test_refusals_of_the_c_abi():
    """Arguments that are checked before a device is looked for."""
    S, INVALID, UNSUPPORTED = ord("s"), 1, 2
    assert status_of("docc_b200_rmsnorm", ord("d"), 1, 8, 1, 8, None, 0, None, 1e-6, None, 1, 0) == INVALID
    assert status_of("docc_b200_rmsnorm", S, -1, 8, 1, 8, None, 0, None, 1e-6, None, 1, 0) == INVALID
    assert status_of("docc_b200_rmsnorm", S, 1, 8, 1, 8, None, 0, None, -1.0, None, 1, 0) == INVALID
    assert status_of("docc_b200_rmsnorm", S, 1, 8, 1, 8, None, 0, None, 1e-6, None, None, 0) == INVALID
    assert status_of("docc_b200_rmsnorm_q8", S, 1, 8, 1, 8, None, 0, None, 1e-6, 64, None, 1, 1, 0) == INVALID
    assert status_of("docc_b200_rope", S, 1, 1, 8, 5, 0, 0, 16, None, 16, 16, 1.0, 16, None, 0) == INVALID
    assert status_of("docc_b200_rope", S, 1, 1, 8, 10, 0, 0, 16, None, 16, 16, 1.0, 16, None, 0) == INVALID
    assert status_of("docc_b200_rope", S, 1, 1, 8, 8, 0, 0, 16, None, None, 16, 1.0, 16, None, 0) == INVALID
    append = lambda page, flags: status_of("docc_b200_rope_append", S, 1, 1, 1, 8, 8, 0, 16, None, 16, None, 16, None, 16, 16, 1.0, 16, None, 16,
                                           None, 16, None, 1, page, 16, flags)
    assert append(0, 0) == INVALID and append(4, 1) == UNSUPPORTED
    attend = lambda prec=S, page=4, cap=0.0, window=0, flags=0: status_of(
        "docc_b200_paged_attention", prec, 1, 1, 1, 8, 1.0, cap, window, 16, None, 16, None, 16, None, 1, page, 16, 1, 1, 16, 16, None, None, None, 0, flags)
    assert attend(prec=ord("d")) == INVALID and attend(page=0) == INVALID and attend(cap=-1.0) == INVALID and attend(window=-1) == INVALID
    assert attend(flags=1) == UNSUPPORTED and attend(cap=float("inf")) == INVALID and attend(cap=float("nan")) == INVALID
    logp = lambda k=0, scale=1.0, prec=S: status_of("docc_b200_token_logprobs", prec, 1, 8, 16, 8, scale, 16, 16, 16, k, 16, 16, 0)
    assert logp(k=9) == INVALID and logp(k=33) == INVALID and logp(k=-1) == INVALID and logp(scale=0.0) == INVALID
    assert logp(scale=float("nan")) == INVALID and logp(prec=ord("d")) == INVALID


@gpu
def test_refusals_with_a_device(rt):
    q = torch.zeros(2, 4, 64, device="cuda")
    cache, table, lengths = torch.zeros(3, 2, 16, 64, device="cuda"), torch.zeros(2, 1, dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda()
    good = dict(q=q, k_cache=cache, v_cache=cache, page_table=table, lengths=lengths)
    assert (ops.paged_attention(**good) == 0).all()
    for change, error in [(dict(lengths=lengths.long()), TypeError), (dict(page_table=table.long()), TypeError), (dict(lengths=lengths[:1]), ValueError),
                          (dict(q=torch.zeros(2, 3, 64, device="cuda")), ValueError), (dict(v_cache=cache[:2]), ValueError),
                          (dict(k_cache=cache.half(), v_cache=cache.half()), ValueError), (dict(q=q.cpu()), TypeError),
                          (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), ValueError), (dict(out=q[0].expand(2, 4, 64)), ValueError),
                          (dict(softcap=-1.0), _lib.DoccB200Error), (dict(window=-1), _lib.DoccB200Error)]:
        with pytest.raises(error):
            ops.paged_attention(**{**good, **change})
    big = torch.zeros(1, 1, 300, device="cuda")
    with pytest.raises(_lib.DoccB200Error) as e:
        ops.paged_attention(big, big[None], big[None], table[:1], lengths[:1])
    assert e.value.status == 2
    with pytest.raises(_lib.DoccB200Error) as e:
        ops.rmsnorm(torch.zeros(1, 40000, device="cuda"))
    assert e.value.status == 2
    with pytest.raises(_lib.DoccB200Error):
        ops.token_logprobs(q[0], torch.zeros(4, dtype=torch.int64).cuda(), k=33)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_of_no_extent(rt, dtype):
    """Empty batches, an empty cache under empty sequences, a table without pages, and no tokens."""
    empty = lambda *s: torch.empty(*s, dtype=dtype, device="cuda")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    i64 = lambda n: torch.zeros(n, dtype=torch.int64, device="cuda")
    assert ops.paged_attention(empty(0, 4, 64), empty(3, 2, 16, 64), empty(3, 2, 16, 64), i32(0, 2), i32(0)).shape == (0, 4, 64)
    q = normal(2, 4, 64, seed=1, dtype=dtype).cuda()
    for pages, most in ((0, 0), (0, 3), (3, 0)):
        out, lse = ops.paged_attention(q, empty(pages, 2, 16, 64), empty(pages, 2, 16, 64), i32(2, most), i32(2), return_lse=True)
        settle()
        assert (out == 0).all() and (lse == -math.inf).all()
    freq = torch.from_numpy(ops.rope_frequencies(64)[0]).cuda()
    cache = torch.zeros(2, 2, 4, 64, dtype=dtype, device="cuda")
    assert ops.rope_append(empty(0, 4, 64), empty(0, 2, 64), empty(0, 2, 64), i64(0), freq, cache, cache.clone(), i64(0)).shape == (0, 4, 64)
    assert ops.rope(empty(0, 4, 64), i64(0), freq).shape == (0, 4, 64) and ops.rope(empty(3, 0, 64), i64(3), freq).shape == (3, 0, 64)
    assert [t.shape for t in ops.token_logprobs(empty(0, 10), i64(0), k=3)] == [(0,), (0,), (0, 3), (0, 3)]
    assert ops.rmsnorm(empty(0, 64)).shape == (0, 64) and ops.rmsnorm(empty(4, 0)).shape == (4, 0)
    assert [t.shape for t in ops.rmsnorm_quant(empty(0, 64), group=128)] == [(0, 64), (0, 1)]
    with pytest.raises(_lib.DoccB200Error):
        ops.token_logprobs(empty(2, 0), i64(2))
    settle()


@gpu
def test_paged_attention_may_write_over_its_query(rt):
    """A split sequence's parts all read the query before the join writes the output."""
    q, kc, vc, table, lengths = paged_problem([5000, 3, 0, 700], 8, 2, 64, 16, torch.bfloat16)
    want = ops.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda())
    over = q.cuda()
    got = ops.paged_attention(over, kc, vc, table.cuda(), lengths.cuda(), out=over)
    settle()
    assert got.data_ptr() == over.data_ptr() and torch.equal(over, want)


@gpu
def test_paged_attention_many_sequences(rt):
    """More sequences than one pass of a warp over the lengths, most of them short."""
    lengths = [(7 * b) % 50 for b in range(150)]
    lengths[77] = 2500
    check_paged(paged_problem(lengths, 2, 1, 64, 8, torch.float16))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 700])
def test_token_logprobs_when_very_many_logits_compete(rt, rows, dtype):
    """Rows in which more logits reach the first bound than are kept at a time: all equal, two values, all but three masked out."""
    vocab = 131072 if rows == 2 else 9000
    x = torch.zeros(rows, vocab, dtype=dtype)
    x[1, ::3] = 1.0
    if rows > 2:
        x[2::7] = -float("inf")
        x[2::7, 4000:4003] = torch.tensor([1.0, 5.0, 1.0], dtype=dtype)
        x[3::7, 1000:] = 2.0
    check_logprobs(x, torch.full((rows,), 4001), 32)
    check_logprobs(x, torch.full((rows,), 4001), 1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_of_rows_full_of_nan(rt, dtype):
    x = normal(3, 30001, seed=3, dtype=dtype)
    x[0, 5000:] = float("nan")
    x[1, 7::2] = float("nan")
    x[2, 1234] = float("inf")
    logp, entropy, top_ids, top_logp = ops.token_logprobs(x.cuda(), torch.tensor([1, 2, 1234]).cuda(), k=4)
    settle()
    assert torch.isnan(logp).all() and torch.isnan(entropy).all() and torch.isnan(top_logp).all()
    assert top_ids[0].tolist() == [5000, 5001, 5002, 5003] and top_ids[1].tolist() == [7, 9, 11, 13] and top_ids[2, 0] == 1234


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,allowed", [(1, 131072, 1), (3, 128001, 3), (40, 50021, 19), (160, 32000, 2), (600, 128000, 5)])
def test_token_logprobs_when_a_mask_leaves_fewer_tokens_than_asked(rt, rows, vocab, allowed, dtype):
    """The masked tokens fill the list in the order of their indices, with a log-probability of -inf."""
    x = torch.full((rows, vocab), -float("inf"), dtype=dtype)
    at = torch.randint(vocab, (rows, allowed), generator=torch.Generator().manual_seed(rows))
    x.scatter_(1, at, normal(rows, allowed, seed=vocab, dtype=dtype))
    check_logprobs(x, at[:, 0], 20)
