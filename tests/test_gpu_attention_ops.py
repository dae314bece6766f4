"""The attention operators (qk_norm.hip, soft_max_rel.hip, diff_attention.hip) against their definitions in 64 bits,
over element types, layouts, odd sizes, strides, masks and empty inputs.

Bounds are per element, from the roundings of each step (u = 2^-24 for a float operation, h = half a step of the
result's type relative to the value, plus half the smallest subnormal step of fp16):
  qk      the norm's factor (rounded once from double) times x times w: 3 u |z|; the rotation as in stx_rope_scaled:
          4 u m (|z0| + |z1|); together 8 u m (|z0| + |z1|). Gradient: dz within 4 u m (|dy0| + |dy1|) = 4 u D; with
          g = w dz, dx = r (g - xh mean(g xh)): each term's roundings, 8 u r (|w| D + |xh| mean(|w| D |xh|)).
          dw: sums of dz xh over n rows in float of at most n / 4 + 64 terms: each partial sum is at most S = sum |D xh|,
          a random walk of sqrt(n) roundings u S / ... bounded by (8 + 4 sqrt(n)) u S.
"""
import math

import pytest

import stx
from test_gpu_layer_ops import F64, TYPES, U, YARN, close, randn, rope_ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ------------------------------------------------------------------------- norms and rotation
def norm_rows(x, w, eps):
    """x, w / sqrt(mean(x^2) + eps) x, and the factor, in 64 bits; w (D,), (H, D) or None."""
    x = x.to(F64)
    r = 1.0 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return x, (x * r if w is None else x * r * w.to(F64)), r


def qk_ref(x, w, pos, eps, n_dims, mode, **setting):
    z = norm_rows(x, w, eps)[1]
    return rope_ref(z, pos, n_dims, mode, **setting)


def qk_back_ref(dy, x, w, pos, eps, n_dims, mode, **setting):
    """dx, dw (per element of a row, unsummed) and the bounds of both."""
    dz, mag = rope_ref(dy.to(F64), pos, n_dims, mode, back=True, **setting)
    mag = torch.where(mag > 0, mag, dz.abs())
    x, _, r = norm_rows(x, w, eps)
    w = 1.0 if w is None else w.to(F64)
    xh, g = x * r, w * dz
    gm = (abs(w) if not isinstance(w, float) else w) * mag
    dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
    return dx, 8 * U * r * (gm + xh.abs() * (gm * xh.abs()).mean(-1, keepdim=True)), dz * xh, (mag * xh).abs()


QK = [
    # B, N, H, Hk, D, n_dims, mode, setting, first position, weights
    (1, 1, 8, 8, 64, 64, 0, {}, 0, "shared"),
    (1, 1, 40, 8, 128, 128, 2, YARN, 131071, "shared"),
    (3, 17, 4, 2, 64, 64, 0, {}, 5, "heads"),
    (2, 33, 4, 1, 128, 96, 2, YARN, 100000, "heads"),
    (2, 70, 32, 8, 128, 96, 2, YARN, 0, "heads"),               # more rows than groups of lanes
    (2, 9, 3, 1, 80, 38, 2, dict(freq_scale=0.25), 1000, "shared"),   # 19 pairs: element by element
    (2, 9, 3, 1, 80, 38, 0, dict(freq_scale=0.25), 1000, "none"),     # the last rotated pair inside a vector
    (2, 9, 3, 1, 80, 40, 2, {}, 3, "heads"),                    # halves of 20: vectors of 8 bytes
    (1, 700, 2, 2, 32, 30, 0, {}, 0, "shared"),
    (2, 5, 2, 1, 33, 32, 0, {}, 7, "shared"),                   # odd rows
    (2, 5, 2, 1, 33, 32, 2, {}, 7, "heads"),
    (2, 5, 1, 1, 2, 2, 0, {}, 7, "shared"),
    (2, 300, 1, 1, 4, 2, 2, {}, 7, "heads"),
    (1, 3, 1, 1, 600, 512, 2, YARN, 40, "shared"),              # rows of several units a lane
    (1, 3, 2, 1, 1024, 1024, 0, {}, 40, "heads"),
    (1, 3, 2, 1, 777, 8, 2, {}, 40, "heads"),                   # the same, element by element
    (1, 5000, 1, 1, 12, 8, 2, dict(attn_factor=1.3), 0, "shared"),    # several tokens a block
]


def qk_inputs(device, dt, shape):
    B, N, H, Hk, D, n_dims, mode, setting, first, kind = shape
    q, k = randn(device, (B, N, H, D), 1, 1.5, dtype=dt), randn(device, (B, N, Hk, D), 2, 0.7, dtype=dt)
    lead = {"none": None, "shared": ((), ()), "heads": ((H,), (Hk,))}[kind]
    wq, wk = (None, None) if lead is None else (randn(device, (*s, D), 3 + i, 0.3, 1.0) for i, s in enumerate(lead))
    return q, k, wq, wk, torch.arange(first, first + N, device=device, dtype=torch.int32), stx.rope_params(n_dims, mode, **setting)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", QK, ids=lambda s: "-".join(str(v) for v in (*s[:7], s[9])))
def test_qk_norm_rope(device, dtype, shape):
    n_dims, mode, setting = shape[5:8]
    q, k, wq, wk, pos, p = qk_inputs(device, TYPES[dtype], shape)
    yq, yk = stx.qk_norm_rope(q, pos, p, wq, k, wk, eps=1e-5)
    for got, x, w in ((yq, q, wq), (yk, k, wk)):
        want, mag = qk_ref(x, w, pos, 1e-5, n_dims, mode, **setting)
        close(got, want, 8 * U * torch.maximum(mag, want.abs()), "qk")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", QK, ids=lambda s: "-".join(str(v) for v in (*s[:7], s[9])))
def test_qk_norm_rope_back(device, dtype, shape):
    B, N, H, Hk, D, n_dims, mode, setting, _, kind = shape
    q, k, wq, wk, pos, p = qk_inputs(device, TYPES[dtype], shape)
    dyq, dyk = randn(device, q.shape, 5, dtype=q.dtype), randn(device, k.shape, 6, dtype=q.dtype)
    dq, dwq, dk, dwk = stx.qk_norm_rope_back(dyq, q, pos, p, wq, dyk, k, wk, eps=1e-5)
    for got, dw, dy, x, w in ((dq, dwq, dyq, q, wq), (dk, dwk, dyk, k, wk)):
        want, bound, dww, dwm = qk_back_ref(dy, x, w, pos, 1e-5, n_dims, mode, **setting)
        close(got, want, bound, "dx")
        if kind == "none":
            assert dw is None
            continue
        dims = (0, 1) if kind == "heads" else (0, 1, 2)
        n = dww.numel() // dw.numel()
        close(dw, dww.sum(dims), (8 + 4 * math.sqrt(n)) * U * dwm.sum(dims), "dw")


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("dtype", TYPES)
def test_qk_slices_and_in_place(device, dtype, mode):
    """q and k as slices of a projection, positions of their own per sequence; in place the same bits, forward and
    backward, and the rest of the projection as it was. One side alone gives what both together do."""
    B, N, H, Hk, D = 3, 21, 4, 2, 64
    qkv = randn(device, (B, N, H + 2 * Hk, D), 3, dtype=TYPES[dtype])
    of = lambda t: (t[:, :, :H], t[:, :, H:H + Hk])  # noqa: E731
    q, k = of(qkv)
    pos = torch.stack([torch.arange(N, device=device) * (b + 1) - 9 for b in range(B)]).to(torch.int32)
    factors = torch.linspace(1.0, 8.0, 24, device=device)
    p = stx.rope_params(48, mode, factors)
    wq, wk = randn(device, (H, D), 4, 0.3, 1.0), randn(device, (Hk, D), 5, 0.3, 1.0)
    yq, yk = stx.qk_norm_rope(q, pos, p, wq, k, wk)
    for got, x, w in ((yq, q, wq), (yk, k, wk)):
        want, mag = qk_ref(x, w, pos, 1e-6, 48, mode, factors=factors)
        close(got, want, 8 * U * torch.maximum(mag, want.abs()), "slices")
    copy = qkv.clone()
    stx.qk_norm_rope(of(copy)[0], pos, p, wq, of(copy)[1], wk, out=of(copy)[0], k_out=of(copy)[1])
    assert torch.equal(of(copy)[0], yq) and torch.equal(of(copy)[1], yk) and torch.equal(copy[:, :, H + Hk:], qkv[:, :, H + Hk:])
    assert torch.equal(stx.qk_norm_rope(q, pos, p, wq), yq) and torch.equal(stx.qk_norm_rope(k, pos, p, wk), yk)
    dy = randn(device, qkv.shape, 6, dtype=TYPES[dtype])
    dq, dwq, dk, dwk = stx.qk_norm_rope_back(of(dy)[0], q, pos, p, wq, of(dy)[1], k, wk)
    alone = stx.qk_norm_rope_back(of(dy)[0], q, pos, p, wq)
    assert torch.equal(alone[0], dq) and alone[2] is None and alone[3] is None
    for into in (dy, qkv):
        copy = into.clone()
        src = (of(copy)[0], of(copy)[1]) if into is dy else of(dy)
        x = of(copy) if into is qkv else (q, k)
        got = stx.qk_norm_rope_back(src[0], x[0], pos, p, wq, src[1], x[1], wk, dq=of(copy)[0], dk=of(copy)[1])
        assert torch.equal(of(copy)[0], dq) and torch.equal(of(copy)[1], dk) and torch.equal(copy[:, :, H + Hk:], into[:, :, H + Hk:])
        assert torch.equal(got[1], dwq) and torch.equal(got[3], dwk)


def test_qk_gradient_against_differences(device):
    """The gradients against central differences of the definition in 64 bits."""
    B, N, H, D, eps = 1, 3, 2, 16, 1e-3
    x, w, dy = randn(device, (B, N, H, D), 1), randn(device, (D,), 2, 0.3, 1.0), randn(device, (B, N, H, D), 3)
    pos = torch.arange(4, 4 + N, device=device, dtype=torch.int32)
    dx, dw, _, _ = stx.qk_norm_rope_back(dy, x, pos, stx.rope_params(12, 2), w, eps=eps)
    f = lambda x, w: float((qk_ref(x, w, pos, eps, 12, 2)[0] * dy.to(F64)).sum())  # noqa: E731
    step = 1e-5
    for t, got in ((x, dx), (w, dw)):
        t64 = t.to(F64)
        for i in range(0, t.numel(), 7):
            d = torch.zeros_like(t64).view(-1)
            d[i] = step
            d = d.view_as(t64)
            diff = (f(t64 + d, w) - f(t64 - d, w) if t is x else f(x, t64 + d) - f(x, t64 - d)) / (2 * step)
            assert abs(float(got.view(-1)[i]) - diff) < 1e-5 * max(1.0, abs(diff))


def test_qk_values_whose_squares_leave_fp32(device):
    for scale in (1e25, 1e-25):
        x = randn(device, (1, 5, 2, 64), 1, scale)
        pos = torch.arange(5, device=device, dtype=torch.int32)
        y = stx.qk_norm_rope(x, pos, stx.rope_params(64), eps=0.0)
        want, mag = qk_ref(x, None, pos, 0.0, 64, 0)
        close(y, want, 8 * U * mag, "range")


def test_qk_empty(device):
    p = stx.rope_params(8)
    w = torch.ones(8, device=device)
    x = torch.empty((2, 0, 3, 8), device=device)
    pos = torch.empty(0, dtype=torch.int32, device=device)
    assert stx.qk_norm_rope(x, pos, p, w).shape == x.shape
    dx, dw, _, _ = stx.qk_norm_rope_back(x, x, pos, p, w)
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros(8, device=device))
