"""The transformer-layer operators (rope.hip, group_norm_cl.hip, gated_ff.hip) against their
definitions in 64 bits, over element types, layouts, odd sizes, strides and empty inputs.

Bounds are per element, from the roundings of each step (u = 2^-24 for a float operation, h = half a
step of the result's type relative to the value, plus half the smallest subnormal step of fp16):
  rope    cos and sin rounded once, one product and one fused operation: 4 u m (|x0| + |x1|).
  norm    x - mean, times rstd, less the mean's rest, times w plus b: 8 u (|xhat w| + |b|) of z; an
          activation's slope is at most 1.13 and its evaluation within 16 u, times 1 + z^2 in the
          tails (the exponent's rounding).
  ff      a dot product of K float terms drifts like a random walk of K roundings of its partial
          sums, each at most S = sum |x w|: 4 sqrt(K) u S. Products and activation as above. In the
          backward pass dg and dv are rounded to the type: h |dg| |w| summed.
Sums over rows are taken in double or as float partial sums and bounded by the sum of the terms'
bounds. Where roundings to the type dominate, the 2-norm is bounded too: independent roundings of
relative size at most h have a root mean square of h / sqrt(3), two layers of them 0.82 h.
"""
import math

import pytest

import stx

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
F64 = torch.float64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = {"none": stx.ACT_NONE, "gelu": stx.ACT_GELU, "silu": stx.ACT_SILU, "sigmoid": stx.ACT_SIGMOID}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def randn(device, shape, seed, scale=1.0, mean=0.0, dtype=torch.float32):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device=device) * scale + mean).to(dtype)


def close(got, want, extra, what):
    """|got - want| <= half a step of got's type at want + extra."""
    assert got.shape == want.shape, what
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -149
    bound = half_step(got.dtype) * (want.abs() + extra) + extra + tiny if got.dtype != F64 else extra
    off = (got.to(F64) - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).max()):.2f} times the bound"


def norm_close(got, want, layers, what):
    if want.numel() < 64 or got.dtype == torch.float32:
        return
    h = half_step(got.dtype) * math.sqrt(layers / 3.0) * 1.2
    assert float((got.to(F64) - want).norm()) <= h * float(want.norm()), what


# ------------------------------------------------------------------------------- rope
def rope_ref(x, pos, n_dims, mode, factors=None, freq_base=10000.0, freq_scale=1.0, n_ctx_orig=0, ext_factor=0.0,
             attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, back=False):
    """(result, |x0| + |x1| of each element's pair times m) in 64 bits; x (B, N, H, D), pos (N,) or (B, N)."""
    f = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731  the ABI's floats
    base, scale, ext, m = f(freq_base), f(freq_scale), f(ext_factor), f(attn_factor)
    i = torch.arange(n_dims // 2, device=x.device, dtype=F64)
    far = base ** (-2.0 * i / n_dims)
    if factors is not None:
        far = far / factors.to(F64)
    freq = scale * far
    if ext:
        d = lambda r: n_dims * math.log(n_ctx_orig / (2 * math.pi * r)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(0.0, math.floor(d(beta_fast))), min(n_dims - 1.0, math.ceil(d(beta_slow)))
        mix = ext * (1.0 - ((i - lo) / max(0.001, hi - lo)).clamp(0, 1))
        freq = scale * far * (1 - mix) + far * mix
        m *= 1.0 + 0.1 * math.log(1.0 / scale)
    theta = pos.to(F64).reshape(-1, x.shape[1], 1, 1) * freq
    c, s = theta.cos() * m, theta.sin() * m * (-1 if back else 1)
    y = x.to(F64, copy=True)
    mag = torch.zeros_like(y)
    a = slice(0, n_dims, 2) if mode == 0 else slice(0, n_dims // 2)
    b = slice(1, n_dims, 2) if mode == 0 else slice(n_dims // 2, n_dims)
    x0, x1 = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = x0 * c - x1 * s, x0 * s + x1 * c
    mag[..., a] = mag[..., b] = abs(m) * (x0.abs() + x1.abs())
    return y, mag


YARN = dict(freq_base=500000.0, freq_scale=0.125, n_ctx_orig=8192, ext_factor=1.0)
ROPE = [
    # B, N, H, Hk, D, n_dims, mode, setting, first position
    (1, 1, 8, 8, 64, 64, 0, {}, 0),
    (1, 1, 40, 8, 128, 128, 2, YARN, 131071),
    (3, 17, 4, 2, 64, 64, 0, {}, 5),
    (2, 33, 4, 1, 128, 96, 2, YARN, 100000),
    (2, 9, 3, 1, 80, 38, 2, dict(freq_scale=0.25), 1000),      # 19 pairs: element by element
    (2, 9, 3, 1, 80, 38, 0, dict(freq_scale=0.25), 1000),      # the last rotated pair inside a vector
    (1, 700, 2, 2, 32, 30, 0, {}, 0),
    (2, 5, 2, 1, 33, 32, 0, {}, 7),                             # odd rows
    (2, 5, 2, 1, 33, 32, 2, {}, 7),
    (2, 5, 1, 1, 2, 2, 0, {}, 7),
    (1, 3, 1, 1, 600, 512, 2, YARN, 40),                        # pairs beyond a block's threads
    (1, 2500, 1, 1, 12, 8, 2, dict(attn_factor=1.3), 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ROPE, ids=lambda s: "-".join(str(v) for v in s[:7]))
@pytest.mark.parametrize("back", [False, True])
def test_rope_scaled(device, dtype, shape, back):
    B, N, H, Hk, D, n_dims, mode, setting, first = shape
    dt = TYPES[dtype]
    q, k = randn(device, (B, N, H, D), 1, dtype=dt), randn(device, (B, N, Hk, D), 2, dtype=dt)
    pos = torch.arange(first, first + N, device=device, dtype=torch.int32)
    p = stx.rope_params(n_dims, mode, **setting)
    call = stx.rope_scaled_back if back else stx.rope_scaled
    yq, yk = call(q, pos, p, k)
    for name, got, x in (("q", yq, q), ("k", yk, k)):
        want, mag = rope_ref(x, pos, n_dims, mode, back=back, **setting)
        close(got, want, 4 * U * mag, name)
    assert torch.equal(yq[..., n_dims:], q[..., n_dims:])


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("dtype", TYPES)
def test_rope_slices_positions_factors_and_in_place(device, dtype, mode):
    """q and k as slices of a projection, positions of their own per sequence (negative ones among them), frequency
    factors; in place the same bits, and the rest of the projection as it was."""
    B, N, H, Hk, D = 3, 21, 4, 2, 64
    qkv = randn(device, (B, N, H + 2 * Hk, D), 3, dtype=TYPES[dtype])
    q, k = qkv[:, :, :H], qkv[:, :, H:H + Hk]
    pos = torch.stack([torch.arange(N, device=device) * (b + 1) - 9 for b in range(B)]).to(torch.int32)
    factors = torch.linspace(1.0, 8.0, 24, device=device)
    p = stx.rope_params(48, mode, factors)
    yq, yk = stx.rope_scaled(q, pos, p, k)
    for got, x in ((yq, q), (yk, k)):
        want, mag = rope_ref(x, pos, 48, mode, factors)
        close(got, want, 4 * U * mag, "slices")
    copy = qkv.clone()
    stx.rope_scaled(copy[:, :, :H], pos, p, copy[:, :, H:H + Hk], copy[:, :, :H], copy[:, :, H:H + Hk])
    assert torch.equal(copy[:, :, :H], yq) and torch.equal(copy[:, :, H:H + Hk], yk)
    assert torch.equal(copy[:, :, H + Hk:], qkv[:, :, H + Hk:])
    one = stx.rope_scaled(q, pos, p)
    assert torch.equal(one, yq)
    # Rows that start off a vector's alignment.
    off = torch.empty(B * N * H * D + 1, dtype=q.dtype, device=device)[1:].view(B, N, H, D)
    off.copy_(q)
    assert torch.equal(stx.rope_scaled(off, pos, p), yq)


def test_rope_matches_rope_ext(device):
    """Without scaling, the rotation of rope_ext, to two float roundings."""
    x = randn(device, (2, 50, 4, 64), 4)
    pos = torch.arange(50, device=device, dtype=torch.int32)
    for mode in (0, 2):
        a = stx.rope_scaled(x, pos, stx.rope_params(64, mode))
        b = stx.rope_ext(x, pos, 64, mode)
        mag = rope_ref(x, pos, 64, mode)[1]
        assert bool(((a - b).abs() <= 6 * U * mag).all())


def test_rope_gradient_by_differences(device):
    """<dy, R x> is linear in x: the gradient is R^T dy, so <dy, R x> = <R^T dy, x>; and R^T R = m^2."""
    x, dy = randn(device, (1, 40, 2, 64), 5), randn(device, (1, 40, 2, 64), 6)
    pos = torch.arange(40, device=device, dtype=torch.int32) * 3000
    p = stx.rope_params(48, 2, **YARN)
    y, dx = stx.rope_scaled(x, pos, p), stx.rope_scaled_back(dy, pos, p)
    a, b = (dy.to(F64) * y.to(F64)).sum(), (dx.to(F64) * x.to(F64)).sum()
    scale = (dy.to(F64) * y.to(F64)).abs().sum()
    assert abs(float(a - b)) <= 16 * U * float(scale)


@pytest.mark.parametrize("shape", [(0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)])
def test_rope_empty(device, shape):
    q = torch.empty(shape, device=device)
    pos = torch.zeros(shape[1], device=device, dtype=torch.int32)
    assert stx.rope_scaled(q, pos, stx.rope_params(64)).shape == shape


# ------------------------------------------------------------------- group norm, channels last
def act_ref(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s, r = torch.sigmoid(z), torch.sigmoid(-z)
    return (z * s, s + z * s * r) if act == "silu" else (s, s * r)


def groups_of(C, G):
    w = -(-C // G)
    return [slice(lo, min(lo + w, C)) for lo in range(0, C, w)]


def norm_ref(x, G, eps, w, b, act, dy=None):
    """Everything about the normalisation of x (B, T, C) in 64 bits, with the bounds of its outputs."""
    x = x.to(F64)
    C = x.shape[2]
    w = torch.ones(C, dtype=F64, device=x.device) if w is None else w.to(F64)
    b = torch.zeros(C, dtype=F64, device=x.device) if b is None else b.to(F64)
    mean, rstd = torch.empty(x.shape[0], len(groups_of(C, G)), dtype=F64, device=x.device), None
    rstd = torch.empty_like(mean)
    xh = torch.empty_like(x)
    for g, ch in enumerate(groups_of(C, G)):
        m = x[..., ch].mean((1, 2))
        r = ((x[..., ch] - m[:, None, None]).square().mean((1, 2)) + eps).rsqrt()
        mean[:, g], rstd[:, g] = m, r
        xh[..., ch] = (x[..., ch] - m[:, None, None]) * r[:, None, None]
    z = xh * w + b
    ez = 8 * U * ((xh * w).abs() + b.abs())
    a, d = act_ref(z, act)
    out = {"y": a, "ey": 1.13 * ez + 16 * U * (1 + z * z) * a.abs() + 2 * U * z.abs(), "stats": torch.stack([mean, rstd], -1)}
    if dy is None:
        return out
    dy = dy.to(F64)
    dz, edz = dy * d, dy.abs() * (ez + 32 * U * (1 + z.abs()) )
    out["db"], out["edb"] = dz.sum((0, 1)), edz.sum((0, 1)) + 4 * U * dz.abs().sum((0, 1))
    out["dw"], out["edw"] = (dz * xh).sum((0, 1)), (edz * xh.abs() + 8 * U * dz.abs() * (xh.abs() + 1)).sum((0, 1))
    dx, edx = torch.empty_like(x), torch.empty_like(x)
    for g, ch in enumerate(groups_of(C, G)):
        n = max(1, x.shape[1] * (ch.stop - ch.start))
        wdz, ewdz = dz[..., ch] * w[ch], edz[..., ch] * w[ch].abs()
        s1, s2 = wdz.sum((1, 2), keepdim=True) / n, (wdz * xh[..., ch]).sum((1, 2), keepdim=True) / n
        e1 = ewdz.sum((1, 2), keepdim=True) / n
        e2 = (ewdz * xh[..., ch].abs() + 8 * U * wdz.abs() * (xh[..., ch].abs() + 1)).sum((1, 2), keepdim=True) / n
        r = rstd[:, g][:, None, None]
        dx[..., ch] = r * (wdz - s1 - xh[..., ch] * s2)
        edx[..., ch] = r * (ewdz + e1 + e2 * xh[..., ch].abs() + 8 * U * (wdz.abs() + s1.abs() + (xh[..., ch] * s2).abs() + s2.abs()))
    out["dx"], out["edx"] = dx, edx
    return out


NORM = [
    # B, T, C, G
    (1, 1, 1, 1), (1, 1, 512, 1), (1, 1, 7, 7), (2, 3, 5, 2), (1, 1344, 512, 1), (3, 85, 48, 1), (2, 101, 96, 4),
    (1, 37, 33, 3),                     # 33 channels, vectors across rows
    (2, 19, 10, 4),                     # groups of 3, 3, 3 and 1
    (4, 57, 383, 1), (1, 130, 1499, 32), (2, 300, 1500, 4), (70, 1, 24, 8), (1, 4001, 3, 1), (1, 999, 2056, 8), (300, 7, 16, 2),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORM, ids=str)
@pytest.mark.parametrize("act", ["none", "gelu", "silu", "sigmoid"])
def test_group_norm_cl(device, dtype, shape, act):
    B, T, C, G = shape
    x = randn(device, (B, T, C), 11, 1.3, 0.4, TYPES[dtype])
    w, b = randn(device, (C,), 12, 0.3, 1.0), randn(device, (C,), 13, 0.3)
    dy = randn(device, (B, T, C), 14, dtype=TYPES[dtype])
    ref = norm_ref(x, G, 1e-5, w, b, act, dy)
    y, stats = stx.group_norm_cl(x, G, 1e-5, w, b, ACTS[act])
    close(y, ref["y"], ref["ey"], "y")
    assert torch.allclose(stats, ref["stats"], rtol=1e-10, atol=1e-13)
    dx, dw, db = stx.group_norm_cl_back(dy, x, stats, G, w, b, ACTS[act])
    close(dx, ref["dx"], ref["edx"], "dx")
    close(dw, ref["dw"], ref["edw"], "dw")
    close(db, ref["db"], ref["edb"], "db")
    again = stx.group_norm_cl_back(dy, x, stats, G, w, b, ACTS[act])
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 40, 300, 300), (1, 2000, 1024, 512), (1, 20, 4096, 4096), (2, 9, 8000, 4000)], ids=str)
def test_group_norm_cl_many_groups(device, dtype, shape):
    """More groups than a block has threads, up to the most."""
    B, T, C, G = shape
    x, dy = (randn(device, (B, T, C), 71 + i, 1.3, 0.4 - 0.4 * i, TYPES[dtype]) for i in range(2))
    w, b = randn(device, (C,), 73, 0.3, 1.0), randn(device, (C,), 74, 0.3)
    ref = norm_ref(x, G, 1e-5, w, b, "silu", dy)
    y, stats = stx.group_norm_cl(x, G, 1e-5, w, b, stx.ACT_SILU)
    close(y, ref["y"], ref["ey"], "y")
    assert torch.allclose(stats, ref["stats"], rtol=1e-10, atol=1e-13)
    dx, dw, db = stx.group_norm_cl_back(dy, x, stats, G, w, b, stx.ACT_SILU)
    close(dx, ref["dx"], ref["edx"], "dx")
    close(dw, ref["dw"], ref["edw"], "dw")
    close(db, ref["db"], ref["edb"], "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C,shift", [(48, 0), (48, 1), (37, 1)])
def test_group_norm_cl_in_place_alignment_and_4d(device, dtype, C, shift):
    """(B, T1, T2, C); in place; data off a vector's alignment; no weight or bias."""
    B, T1, T2, G = 2, 9, 5, 3
    dt = TYPES[dtype]
    buf = torch.zeros(B * T1 * T2 * C + shift + 8, device=device, dtype=dt)
    x = buf[shift:shift + B * T1 * T2 * C].view(B, T1, T2, C)
    x.copy_(randn(device, (B, T1, T2, C), 15, dtype=dt))
    ref = norm_ref(x.reshape(B, T1 * T2, C), G, 1e-5, None, None, "silu")
    y, _ = stx.group_norm_cl(x, G, act=stx.ACT_SILU)
    close(y.reshape(B, T1 * T2, C), ref["y"], ref["ey"], "y")
    stx.group_norm_cl(x, G, act=stx.ACT_SILU, out=x)
    assert torch.equal(x, y)
    assert not bool(buf[:shift].any()) and not bool(buf[shift + x.numel():].any())
    # dx over dy.
    dy = randn(device, x.shape, 16, dtype=dt)
    x = randn(device, x.shape, 17, dtype=dt)
    _, stats = stx.group_norm_cl(x, G)
    dx, dw, db = stx.group_norm_cl_back(dy, x, stats, G)
    stx.group_norm_cl_back(dy, x, stats, G, dx=dy)
    assert torch.equal(dx, dy)


def test_group_norm_cl_large_mean_and_constant_rows(device):
    """Mean 1000 times the deviation: the float roundings stay those of x - mean. A constant slice has variance 0."""
    x = randn(device, (2, 400, 32), 18, 1.0, 1000.0)
    x[1] = 3.25
    ref = norm_ref(x, 2, 1e-5, None, None, "none")
    y, stats = stx.group_norm_cl(x, 2)
    close(y, ref["y"], ref["ey"], "y")
    assert not bool(y[1].any()) and bool((stats[1, :, 0] == 3.25).all())


def test_group_norm_cl_nan_and_inf_stay_in_their_group(device):
    x = randn(device, (2, 50, 12), 19)
    x[0, 7, 5], x[1, 3, 0] = float("nan"), float("inf")
    y, _ = stx.group_norm_cl(x, 3)                       # groups of 4 channels
    assert bool(y[0, :, 4:8].isnan().all()) and bool(y[1, :, :4].isnan().any())
    rest = torch.ones(2, 12, dtype=torch.bool, device=device)
    rest[0, 4:8], rest[1, :4] = False, False
    assert bool(y.permute(0, 2, 1)[rest].isfinite().all())


@pytest.mark.parametrize("shape", [(0, 5, 16), (3, 0, 16)])
def test_group_norm_cl_empty(device, shape):
    x = torch.empty(shape, device=device)
    y, stats = stx.group_norm_cl(x, 4, 1e-4)
    assert y.shape == shape
    assert bool((stats[..., 0] == 0).all()) and bool((stats[..., 1] == 1 / math.sqrt(1e-4)).all())
    dw, db = (torch.full((16,), 7.0, device=device) for _ in range(2))
    stx.group_norm_cl_back(x, x, stats, 4, dweight=dw, dbias=db)
    assert not bool(dw.any()) and not bool(db.any())


def test_group_norm_cl_matches_group_norm(device):
    """The same normalisation as stx.group_norm of the transposed tensor (fp32, affine, GELU)."""
    C, T = 48, 3001
    x = randn(device, (1, T, C), 20)
    w, b = randn(device, (C,), 21, 0.3, 1.0), randn(device, (C,), 22)
    y, _ = stx.group_norm_cl(x, 1, 1e-5, w, b, stx.ACT_GELU)
    first = stx.group_norm(x[0].t().contiguous().view(C, 1, T), 1, 1e-5, w.view(C, 1, 1), b.view(C, 1, 1), gelu=True)
    ref = norm_ref(x, 1, 1e-5, w, b, "gelu")
    close(first.view(C, T).t()[None], ref["y"], ref["ey"], "group_norm")
    close(y, ref["y"], ref["ey"], "group_norm_cl")


# ---------------------------------------------------------------------------- gated block
def ff_ref(x, wg, wv, act, bg, bv, dh=None):
    """The block in 64 bits with the bounds of its outputs; x (M, K)."""
    dt = x.dtype
    x, wg, wv = (t.to(F64) for t in (x, wg, wv))
    M, K = x.shape
    N = wg.shape[0]
    mm = lambda a, b: torch.mm(a.contiguous(), b.contiguous())  # noqa: E731
    g, v = mm(x, wg.t()), mm(x, wv.t())
    walk = 4 * math.sqrt(K) * U
    eg, ev = walk * mm(x.abs(), wg.abs().t()), walk * mm(x.abs(), wv.abs().t())
    if bg is not None:
        g, eg = g + bg.to(F64), eg + U * bg.to(F64).abs()
    if bv is not None:
        v, ev = v + bv.to(F64), ev + U * bv.to(F64).abs()
    eg, ev = eg + U * g.abs(), ev + U * v.abs()
    a, d = act_ref(g, act)
    ea = 1.13 * eg + 16 * U * (1 + g * g) * a.abs() + 2 * U * g.abs()
    out = {"h": a * v, "eh": ea * v.abs() + a.abs() * ev + 2 * U * (a * v).abs()}
    if dh is None:
        return out
    dh, h = dh.to(F64), half_step(dt)
    ed = eg + 16 * U * (1 + g.abs())                       # slopes of the slopes are at most 0.8
    dg, dv = dh * v * d, dh * a
    edg = dh.abs() * (ev * d.abs() + v.abs() * ed) + 4 * U * dg.abs()
    edv = dh.abs() * ea + 4 * U * dv.abs()
    sums = max(1, M)
    out["dbg"], out["edbg"] = dg.sum(0), edg.sum(0) + 4 * math.sqrt(sums) * U * dg.abs().sum(0)
    out["dbv"], out["edbv"] = dv.sum(0), edv.sum(0) + 4 * math.sqrt(sums) * U * dv.abs().sum(0)
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    fg, fv = edg + h * dg.abs() + tiny, edv + h * dv.abs() + tiny
    walk2, walk3 = 4 * math.sqrt(2 * N) * U, 4 * math.sqrt(sums) * U
    out["dx"] = mm(dg, wg) + mm(dv, wv)
    out["edx"] = mm(fg + walk2 * dg.abs(), wg.abs()) + mm(fv + walk2 * dv.abs(), wv.abs())
    out["dwg"], out["edwg"] = mm(dg.t(), x), mm((fg + walk3 * dg.abs()).t(), x.abs())
    out["dwv"], out["edwv"] = mm(dv.t(), x), mm((fv + walk3 * dv.abs()).t(), x.abs())
    return out


FF = [
    # M, K, N
    (1, 8, 1), (1, 1, 1), (1, 384, 1536), (1, 1000, 77), (16, 384, 100), (17, 65, 33), (33, 129, 50), (64, 512, 256), (65, 512, 256),
    (65, 7, 9), (128, 64, 64), (129, 72, 65), (200, 384, 200), (300, 333, 301), (777, 512, 130), (130, 2055, 40), (1500, 40, 24),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", FF, ids=str)
@pytest.mark.parametrize("act", ["none", "gelu", "silu", "sigmoid"])
def test_gated_ff(device, dtype, shape, act):
    M, K, N = shape
    dt = TYPES[dtype]
    x = randn(device, (M, K), 31, dtype=dt)
    wg, wv = (randn(device, (N, K), 32 + i, K ** -0.5, dtype=dt) for i in range(2))
    bias = M % 2 == 1
    bg, bv = (randn(device, (N,), 34, 0.2), randn(device, (N,), 35, 0.2)) if bias else (None, None)
    dh = randn(device, (M, N), 36, dtype=dt)
    ref = ff_ref(x, wg, wv, act, bg, bv, dh)
    h = stx.gated_ff(x, wg, wv, ACTS[act], bg, bv)
    close(h, ref["h"], ref["eh"], "h")
    norm_close(h, ref["h"], 1, "h")
    dx, dwg, dwv, dbg, dbv = stx.gated_ff_back(dh, x, wg, wv, ACTS[act], bg, bv)
    for name, got in (("dx", dx), ("dwg", dwg), ("dwv", dwv)):
        close(got, ref[name], ref["e" + name], name)
        norm_close(got, ref[name], 2, name)
    if bias:
        close(dbg, ref["dbg"], ref["edbg"], "dbg")
        close(dbv, ref["dbv"], ref["edbv"], "dbv")
    else:
        assert dbg is None and dbv is None
    again = stx.gated_ff_back(dh, x, wg, wv, ACTS[act], bg, bv)
    assert torch.equal(dx, again[0]) and torch.equal(dwg, again[1]) and torch.equal(dwv, again[2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(5000, 392, 1030), (2600, 1160, 2056), (9001, 128, 96)], ids=str)
def test_gated_ff_large(device, dtype, shape):
    """The larger tiles, several of them a block, with edges in every direction and reductions split or not."""
    M, K, N = shape
    dt = TYPES[dtype]
    x, dh = randn(device, (M, K), 37, dtype=dt), randn(device, (M, N), 38, dtype=dt)
    wg, wv = (randn(device, (N, K), 39 + i, K ** -0.5, dtype=dt) for i in range(2))
    bg, bv = randn(device, (N,), 34, 0.2), randn(device, (N,), 35, 0.2)
    ref = ff_ref(x, wg, wv, "sigmoid", bg, bv, dh)
    h = stx.gated_ff(x, wg, wv, stx.ACT_SIGMOID, bg, bv)
    close(h, ref["h"], ref["eh"], "h")
    norm_close(h, ref["h"], 1, "h")
    for name, got in zip(("dx", "dwg", "dwv", "dbg", "dbv"), stx.gated_ff_back(dh, x, wg, wv, stx.ACT_SIGMOID, bg, bv)):
        close(got, ref[name], ref["e" + name], name)
        if not name.startswith("db"):
            norm_close(got, ref[name], 2, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [5, 150])
def test_gated_ff_strides_and_token_dims(device, dtype, M):
    """Rows of larger buffers (x, weights, dh and every output), at odd offsets; token dimensions; the bytes between
    rows as they were."""
    K, N, dt = 96, 72, TYPES[dtype]
    wide = lambda r, c, seed: randn(device, (r, c + 13), seed, dtype=dt)[:, 3:3 + c]  # noqa: E731
    x, wg, wv, dh = wide(M, K, 41), wide(N, K, 42), wide(N, K, 43), wide(M, N, 44)
    ref = ff_ref(x, wg, wv, "silu", None, None, dh)
    room = [torch.full((r, c + 11), 5.0, device=device, dtype=dt) for r, c in ((M, N), (M, K), (N, K), (N, K))]
    outs = [t[:, 2:2 + c] for t, c in zip(room, (N, K, K, K))]
    stx.gated_ff(x, wg, wv, stx.ACT_SILU, out=outs[0])
    stx.gated_ff_back(dh, x, wg, wv, stx.ACT_SILU, dx=outs[1], dw_gate=outs[2], dw_value=outs[3])
    for name, got in zip(("h", "dx", "dwg", "dwv"), outs):
        close(got, ref[name], ref["e" + name], name)
    for t, c in zip(room, (N, K, K, K)):
        assert bool((t[:, :2] == 5).all()) and bool((t[:, 2 + c:] == 5).all())
    x3 = x.contiguous().view(5, M // 5, K)
    assert torch.equal(stx.gated_ff(x3, wg, wv, stx.ACT_SILU).view(M, N), stx.gated_ff(x, wg, wv, stx.ACT_SILU))


def test_gated_ff_few_and_many_tokens_agree(device):
    """The same rows whether 64 or 65 tokens are given (other kernels): within both bounds."""
    x = randn(device, (65, 512), 51, dtype=torch.bfloat16)
    wg, wv = (randn(device, (200, 512), 52 + i, 512 ** -0.5, dtype=torch.bfloat16) for i in range(2))
    ref = ff_ref(x, wg, wv, "gelu", None, None)
    for m in (1, 15, 16, 31, 32, 63, 64, 65):
        close(stx.gated_ff(x[:m], wg, wv, stx.ACT_GELU), ref["h"][:m], ref["eh"][:m], f"{m} tokens")


def test_gated_ff_is_glu_of_a_linear_layer(device):
    """stx.glu of the two products side by side (value first), fp32."""
    x = randn(device, (70, 64), 54)
    wg, wv = randn(device, (40, 64), 55, 0.125), randn(device, (40, 64), 56, 0.125)
    both = torch.cat([x @ wv.t(), x @ wg.t()], 1)
    ref = ff_ref(x, wg, wv, "sigmoid", None, None)
    close(stx.glu(both, 0), ref["h"], ref["eh"] + 1e-6 * ref["h"].abs(), "glu")
    close(stx.gated_ff(x, wg, wv), ref["h"], ref["eh"], "gated_ff")


def test_gated_ff_no_tokens(device):
    x, w = torch.empty(0, 24, device=device), randn(device, (8, 24), 57)
    assert stx.gated_ff(x, w, w).shape == (0, 8)
    full = [torch.full((8, 24), 3.0, device=device) for _ in range(2)] + [torch.full((8,), 3.0, device=device) for _ in range(2)]
    stx.gated_ff_back(torch.empty(0, 8, device=device), x, w, w.clone(), dw_gate=full[0], dw_value=full[1], db_gate=full[2], db_value=full[3])
    assert not any(bool(t.any()) for t in full)


def test_gated_ff_nonfinite_rows_stay_rows(device):
    """A NaN or infinite token spoils its own row only, in both kernels, and K's padding adds nothing."""
    for m in (20, 100):
        x = randn(device, (m, 40), 58, dtype=torch.bfloat16)
        wg, wv = (randn(device, (24, 40), 59 + i, 0.2, dtype=torch.bfloat16) for i in range(2))
        clean = stx.gated_ff(x, wg, wv)
        x[3, 39], x[m - 1, 0] = float("nan"), float("inf")
        h = stx.gated_ff(x, wg, wv)
        keep = [i for i in range(m) if i not in (3, m - 1)]
        assert bool(h[3].isnan().all()) and torch.equal(h[keep], clean[keep])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gated_ff_partial_gradients(device, dtype):
    """Only some of the outputs through the C ABI: the same bits as with all of them."""
    M, K, N, dt = 150, 48, 40, TYPES[dtype]
    x, dh = randn(device, (M, K), 61, dtype=dt), randn(device, (M, N), 62, dtype=dt)
    wg, wv = (randn(device, (N, K), 63 + i, 0.2, dtype=dt) for i in range(2))
    bg, bv = randn(device, (N,), 65), randn(device, (N,), 66)
    full = stx.gated_ff_back(dh, x, wg, wv, stx.ACT_GELU, bg, bv)
    need = stx.gated_ff_back_workspace_size(M, K, N, dt)
    for pick in ([0], [1, 2], [3], [4], [0, 4]):
        out = [torch.empty_like(t) for t in full]
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        d = [stx._typed(t, x, "t") for t in (dh, x, wg, wv)]
        o = [stx._typed(out[i], x, "o") if i in pick else None for i in range(3)]
        f = [out[i].data_ptr() if i in pick else None for i in (3, 4)]
        stx.check(stx.lib().stx_gated_ff_back(*d, stx._type(x), bg.data_ptr(), bv.data_ptr(), stx.ACT_GELU, *o, *f,
                                              ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
        for i in pick:
            assert torch.equal(out[i], full[i]), i


# --------------------------------------------------------------------------- together, graphs
def layer(x, p, pos, rope, heads):
    """One transformer layer's forward pass, half precision where the operators have it."""
    B, N, D = x.shape
    qkv = (stx.rms_norm(x.float(), 1e-6, p["gamma"]).to(x.dtype) @ p["wqkv"].t()).view(B, N, 3 * heads, D // heads)
    q, k = stx.rope_scaled(qkv[:, :, :heads], pos, rope, qkv[:, :, heads:2 * heads])
    v = qkv[:, :, 2 * heads:]
    score = torch.matmul(q.transpose(1, 2).float().contiguous(), k.permute(0, 2, 3, 1).float().contiguous())
    prob = stx.soft_max_ext(score, (D // heads) ** -0.5)
    o = stx.merge_heads(torch.matmul(prob, v.transpose(1, 2).float().contiguous()))
    x = x + o.reshape(B, N, D).to(x.dtype)
    h = stx.gated_ff(x, p["wg"], p["wv"], stx.ACT_SILU, p["bg"], p["bv"])
    y, _ = stx.group_norm_cl(x + h @ p["wo"].t(), 1, 1e-5, p["w"], p["b"], stx.ACT_NONE)
    return y


def test_layer_together(device):
    """rope, attention, the gated block and the token norm one after another, against the layer in 64 bits. Six roundings to
    bf16 lie one after another (qkv, q and k, the sums, h, the projection, y), of which the last is relative to
    the output and the others pass through layers of gain about 1: 6 h in the 2-norm."""
    B, N, D, F, heads, dt = 2, 75, 128, 192, 4, torch.bfloat16
    r = lambda *s, seed, scale=1.0, t=dt: randn(device, s, seed, scale, dtype=t)  # noqa: E731
    p = {"gamma": r(D, seed=71, t=torch.float32).abs(), "wqkv": r(3 * D, D, seed=72, scale=D ** -0.5), "wg": r(F, D, seed=73, scale=D ** -0.5),
         "wv": r(F, D, seed=74, scale=D ** -0.5), "bg": r(F, seed=75, t=torch.float32), "bv": r(F, seed=76, t=torch.float32),
         "wo": r(D, F, seed=77, scale=F ** -0.5), "w": r(D, seed=78, t=torch.float32), "b": r(D, seed=79, t=torch.float32)}
    x = r(B, N, D, seed=80)
    pos = torch.arange(N, device=device, dtype=torch.int32)
    got = layer(x, p, pos, stx.rope_params(D // heads, 0), heads)
    x, p = x.to(F64).cpu(), {n: t.to(F64).cpu() for n, t in p.items()}
    a = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * p["gamma"]
    qkv = (a @ p["wqkv"].t()).view(B, N, 3 * heads, D // heads)
    q, k = (rope_ref(qkv[:, :, i * heads:(i + 1) * heads], pos.cpu(), D // heads, 0)[0].transpose(1, 2) for i in range(2))
    prob = torch.softmax(q @ k.transpose(2, 3) * (D // heads) ** -0.5, -1)
    x = x + (prob @ qkv[:, :, 2 * heads:].transpose(1, 2)).transpose(1, 2).reshape(B, N, D)
    h = ff_ref(x.reshape(-1, D), p["wg"], p["wv"], "silu", p["bg"], p["bv"])["h"].view(B, N, F)
    want = norm_ref(x + h @ p["wo"].t(), 1, 1e-5, p["w"], p["b"], "none")["y"]
    assert float((got.cpu().to(F64) - want).norm()) <= 6 * half_step(dt) * float(want.norm())


def test_graph_replays_and_streams(device):
    """A captured forward and backward run of the three operators, replayed on new data with eager calls between, on a
    stream of its own: the eager results each time."""
    B, N, D, F, dt = 2, 90, 64, 96, torch.bfloat16
    x, dy = randn(device, (B, N, D), 91, dtype=dt), randn(device, (B, N, D), 92, dtype=dt)
    dh = randn(device, (B, N, F), 93, dtype=dt)
    wg, wv = (randn(device, (F, D), 94 + i, 0.125, dtype=dt) for i in range(2))
    w, b = randn(device, (D,), 96), randn(device, (D,), 97)
    pos = torch.arange(N, device=device, dtype=torch.int32)
    p = stx.rope_params(16, 2)

    def step(s=None):
        q = stx.rope_scaled(x.view(B, N, 4, 16), pos, p, stream=s).view(B, N, D)
        y, stats = stx.group_norm_cl(q, 4, 1e-5, w, b, stx.ACT_GELU, stream=s)
        h = stx.gated_ff(y, wg, wv, stx.ACT_SILU, stream=s)
        g = stx.gated_ff_back(dh, y, wg, wv, stx.ACT_SILU, stream=s)
        d = stx.group_norm_cl_back(g[0], q, stats, 4, w, b, stx.ACT_GELU, stream=s)
        return [h, *g[:3], *d, stx.rope_scaled_back(d[0].view(B, N, 4, 16), pos, p, stream=s)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(s)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step(s)
    torch.cuda.synchronize()
    for rep in range(4):
        x.copy_(randn(device, (B, N, D), 100 + rep, 1.0 + rep, dtype=dt))
        dh.copy_(randn(device, (B, N, F), 200 + rep, dtype=dt))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), rep


def test_differences(device):
    """Gradients of a scalar of the norm and the block, fp32 against central differences in 64 bits of the definitions."""
    M, K, N = 70, 24, 18
    x, dh = randn(device, (M, K), 301), randn(device, (M, N), 302)
    wg, wv = randn(device, (N, K), 303, 0.3), randn(device, (N, K), 304, 0.3)
    bg, bv = randn(device, (N,), 305), randn(device, (N,), 306)
    got = stx.gated_ff_back(dh, x, wg, wv, stx.ACT_GELU, bg, bv)
    args = [t.to(F64) for t in (x, wg, wv, bg, bv)]
    loss = lambda a: float((ff_ref(*a[:3], "gelu", *a[3:])["h"] * dh.to(F64)).sum())  # noqa: E731
    step = 1e-5
    for i, g in enumerate(got):
        d = randn(device, args[i].shape, 310 + i).to(F64)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step * d, args[i] - step * d
        slope = (loss(up) - loss(down)) / (2 * step)
        assert abs(slope - float((g.to(F64) * d).sum())) <= 1e-5 * float((g.to(F64) * d).abs().sum()), i
    x, dy = randn(device, (2, 30, 12), 321), randn(device, (2, 30, 12), 322)
    w, b = randn(device, (12,), 323), randn(device, (12,), 324)
    _, stats = stx.group_norm_cl(x, 3, 1e-5, w, b, stx.ACT_SILU)
    got = stx.group_norm_cl_back(dy, x, stats, 3, w, b, stx.ACT_SILU)
    args = [t.to(F64) for t in (x, w, b)]
    loss = lambda a: float((norm_ref(a[0], 3, 1e-5, a[1], a[2], "silu")["y"] * dy.to(F64)).sum())  # noqa: E731
    for i, g in enumerate(got):
        d = randn(device, args[i].shape, 330 + i).to(F64)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step * d, args[i] - step * d
        slope = (loss(up) - loss(down)) / (2 * step)
        assert abs(slope - float((g.to(F64) * d).sum())) <= 1e-5 * float((g.to(F64) * d).abs().sum()), i


# ------------------------------------------------------------------- far offsets, shared devices
def test_offsets_past_32_bits(device):
    """Elements and bytes beyond 2^32 in every operator: the last rows against the definition."""
    dt = torch.bfloat16
    q = torch.zeros((1, 70000, 512, 64), dtype=dt, device=device)                  # 2.3e9 elements, 4.6 GB
    q[:, -3:] = randn(device, (1, 3, 512, 64), 401, dtype=dt)
    pos = torch.arange(70000, device=device, dtype=torch.int32)
    y = stx.rope_scaled(q, pos, stx.rope_params(64), out=q.clone())
    want, mag = rope_ref(q[:, -3:], pos[-3:], 64, 0)
    close(y[:, -3:], want, 4 * U * mag, "rope")
    del q, y
    x = torch.zeros((2, 1100000, 1024), dtype=dt, device=device)                   # the second slice starts past 2^31 bytes
    x[1, ::1000] = randn(device, (1100, 1024), 402, dtype=dt)
    y, stats = stx.group_norm_cl(x, 4, act=stx.ACT_SILU)
    assert not bool(y[0].any())
    part = x[1, ::1000].to(F64).view(1100, 4, 256)
    n = 1100000 * 256
    mean = part.sum((0, 2)) / n
    var = part.square().sum((0, 2)) / n - mean * mean
    assert torch.allclose(stats[1], torch.stack([mean, (var + 1e-5).rsqrt()], -1), rtol=1e-10, atol=1e-13)
    z = (part[-3:] - mean[:, None]) * (var + 1e-5).rsqrt()[:, None]
    close(y[1, ::1000][-3:], (z * torch.sigmoid(z)).view(3, 1024), 64 * U * (1 + z.abs()).view(3, 1024), "norm")
    dx, dw, db = stx.group_norm_cl_back(x, x, stats, 4, act=stx.ACT_SILU, dx=y)
    ref = norm_ref(x[1:, ::1000], 4, 1e-5, None, None, "silu", x[1:, ::1000])      # the other rows of dy are 0
    s = (part - mean[:, None]) * (var + 1e-5).rsqrt()[:, None]
    sg = torch.sigmoid(s)
    dz = part * (sg + s * sg * (1 - sg))
    close(db, dz.sum(0).reshape(1024), (64 * U * (1 + s.abs()) * part.abs()).sum(0).reshape(1024), "db")
    assert ref["dx"].shape == (1, 1100, 1024) and bool(dx[1].isfinite().all())
    del x, y, dx
    M, K, N = 600000, 40, 4096                                                     # out: 2.5e9 elements
    x = torch.zeros((M, K), dtype=dt, device=device)
    x[-70:] = randn(device, (70, K), 403, dtype=dt)
    wg, wv = (randn(device, (N, K), 404 + i, K ** -0.5, dtype=dt) for i in range(2))
    h = stx.gated_ff(x, wg, wv, stx.ACT_SILU)
    ref = ff_ref(x[-70:], wg, wv, "silu", None, None, randn(device, (70, N), 406, dtype=dt))
    close(h[-70:], ref["h"], ref["eh"], "h")
    assert not bool(h[:1000].any())
    h.zero_()
    h[-70:] = randn(device, (70, N), 406, dtype=dt)                               # as dh: the other tokens add nothing
    dx, dwg, dwv, _, _ = stx.gated_ff_back(h, x, wg, wv, stx.ACT_SILU)
    close(dx[-70:], ref["dx"], ref["edx"], "dx")
    assert not bool(dx[:1000].any())
    close(dwg, ref["dwg"], ref["edwg"], "dwg")
    close(dwv, ref["dwv"], ref["edwv"], "dwv")


def test_two_streams_at_once(device):
    """Calls of the same operators on two streams, each with its own workspace, many times over: each stream's results."""
    x = [randn(device, (3, 501, 96), 411 + i, dtype=torch.bfloat16) for i in range(2)]
    dh = [randn(device, (3, 501, 160), 413 + i, dtype=torch.bfloat16) for i in range(2)]
    wg, wv = (randn(device, (160, 96), 415 + i, 0.1, dtype=torch.bfloat16) for i in range(2))

    def step(i, s=None):
        y, stats = stx.group_norm_cl(x[i], 8, act=stx.ACT_GELU, stream=s)
        return [y, *stx.group_norm_cl_back(x[i], x[i], stats, 8, act=stx.ACT_GELU, stream=s),
                *stx.gated_ff_back(dh[i], y, wg, wv, stx.ACT_SILU, stream=s)[:3]]

    want = [[t.clone() for t in step(i)] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i, s))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for run in got[i] for a, b in zip(run, want[i]))


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_over_the_input(device, dtype):
    """group_norm_cl_back with dx in x's memory gives the same bits."""
    x, dy = (randn(device, (3, 211, 40), 81 + i, dtype=TYPES[dtype]) for i in range(2))
    w = randn(device, (40,), 83, 0.3, 1.0)
    _, stats = stx.group_norm_cl(x, 5, weight=w, act=stx.ACT_SILU)
    want = stx.group_norm_cl_back(dy, x, stats, 5, w, act=stx.ACT_SILU)
    got = stx.group_norm_cl_back(dy, x, stats, 5, w, act=stx.ACT_SILU, dx=x)
    assert got[0] is x and all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [9, 200])
def test_gated_ff_of_one_row_for_every_token(device, dtype, M):
    """x and dh broadcast (a row stride of 0): the bits of the same rows written out."""
    row, dh = (randn(device, (1, n), 84 + n, dtype=TYPES[dtype]) for n in (48, 24))
    wg, wv = (randn(device, (24, 48), 86 + i, 0.2, dtype=TYPES[dtype]) for i in range(2))
    x, g = row.expand(M, 48), dh.expand(M, 24)
    assert x.stride(0) == 0
    assert torch.equal(stx.gated_ff(x, wg, wv), stx.gated_ff(x.contiguous(), wg, wv))
    dx = torch.empty(M, 48, device=device, dtype=TYPES[dtype])
    got = stx.gated_ff_back(g, x, wg, wv, dx=dx)
    want = stx.gated_ff_back(g.contiguous(), x.contiguous(), wg, wv)
    assert all(torch.equal(p, q) for p, q in zip(got[:3], want[:3]))
