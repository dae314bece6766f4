"""The attention operators (qk_norm.hip, soft_max_rel.hip, diff_attention.hip) against their definitions in 64 bits,
over element types, layouts, odd sizes, strides, masks and empty inputs.

Bounds are per element, from the roundings of each step (u = 2^-24 for a float operation, h = half a step of the
result's type relative to the value, plus half the smallest subnormal step of fp16):
  qk      the norm's factor (rounded once from double) times x times w: 3 u |z|; the rotation as in stx_rope_scaled:
          4 u m (|z0| + |z1|); together 8 u m (|z0| + |z1|). Gradient: dz within 4 u m (|dy0| + |dy1|) = 4 u D; with
          g = w dz, dx = r (g - xh mean(g xh)): each term's roundings, 8 u r (|w| D + |xh| mean(|w| D |xh|)).
          dw: sums of dz xh over n rows in float of at most n / 4 + 64 terms: each partial sum is at most S = sum |D xh|,
          a random walk of sqrt(n) roundings u S / ... bounded by (8 + 4 sqrt(n)) u S.
  rel     an exponent has the roundings of the fused product and bias, of the difference to the row's largest, which is
          of twice their size, and of log2e and the product with it: 5 u (|scale x| + |bias|); at most 5 u Z relative to
          each exponential, Z the row's largest |scale x| + |bias|, as much of their sum, 2 u of the hardware's 2^y each,
          and of the sum a rounding for each of a lane's terms and 16 of the tree. Backward: products and sums are in
          double, so one rounding to float and one to the type; the table's sums one.
  diff    a score is a sum of D float products, off by at most (D + 8) u Z with Z = scale sum |q k|, and so, relative to
          itself, is each exponential, as is their sum: 2 (D + 8) u Z; P is rounded to the type (h) and multiplied by v
          in float, a random walk of 4 sqrt(N) u; in all, of A = sum P |v|, for each map. Backward: see the test.
"""
import math

import pytest

import stx
from test_gpu_layer_ops import F64, TYPES, U, YARN, close, half_step, norm_close, randn, rope_ref

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
    (2, 9, 3, 1, 80, 38, 2, dict(freq_scale=0.25), 1000, "shared"),   # 19 pairs: vectors over the halves' ends
    (1, 9, 2, 1, 16, 2, 2, {}, 3, "heads"),                     # both ends in one vector
    (2, 7, 2, 1, 8, 6, 2, {}, 3, "shared"),
    (1, 9, 3, 1, 96, 46, 2, YARN, 1150, "heads"),
    (1, 3, 1, 1, 600, 502, 2, YARN, 40, "shared"),
    (1, 3, 2, 1, 1024, 1022, 2, {}, 40, "heads"),
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


# ------------------------------------------------------------------ softmax with a position bias
def edges_of(n_buckets, distance, both):
    """(buckets of a side, exact ones, first distance of each of the others), in whole numbers."""
    n = n_buckets // 2 if both else n_buckets
    near = n // 2
    m = n - near
    first = []
    for k in range(m):
        d = near
        while d ** m < near ** (m - k) * distance ** k:
            d += 1
        first.append(d)
    return n, near, first


def buckets_ref(rel, n_buckets, distance, both):
    n, near, first = edges_of(n_buckets, distance, both)
    d = rel.abs() if both else (-rel).clamp(min=0)
    k = d.clamp(max=near)
    for i, edge in enumerate(first):
        k = torch.where(d >= edge, near + i, k)
    return torch.where((rel > 0) & both, k + n, k)


def seen_ref(B, M, N, lengths, starts, causal, device):
    """Which keys each query sees, and key less query position, (B, M, N)."""
    start = torch.zeros(B, device=device, dtype=torch.int64) if starts is None else starts.long()
    end = torch.full((B,), N, device=device) if lengths is None else lengths.long()
    j = torch.arange(N, device=device)
    rel = j - (torch.arange(M, device=device)[:, None] + start[:, None, None])
    mask = (j < end[:, None, None]).expand(B, M, N)
    return (mask & (rel <= 0) if causal else mask), rel


REL = [
    # B, H, M, N, n_buckets, max_distance, both, causal, masks
    (1, 1, 1, 1, 32, 128, True, False, None),
    (8, 8, 1, 801, 32, 128, False, True, "ragged"),
    (2, 3, 60, 60, 32, 128, True, False, None),               # several rows a wave
    (2, 3, 61, 7, 8, 20, True, True, "ragged"),
    (2, 2, 130, 131, 4, 3, True, False, "ragged"),
    (3, 2, 77, 513, 16, 50, False, False, "ragged"),          # later keys all in bucket 0
    (1, 2, 801, 801, 32, 128, True, False, None),
    (2, 1, 90, 1100, 64, 1000, True, False, "ragged"),        # reach beyond most keys
    (1, 2, 40, 2049, 32, 128, False, True, None),
    (1, 1, 9, 4100, 256, 2048, True, False, None),
    (1, 1, 5, 8200, 32, 128, True, False, "ragged"),
    (1, 2, 3, 17001, 32, 128, True, True, "ragged"),          # rows read twice
    (1, 1, 300, 33, 2, 2, False, True, None),
]


def rel_inputs(device, dt, shape):
    B, H, M, N, nb, dist, both, causal, masks = shape
    x = randn(device, (B, H, M, N), 1, 6.0, dtype=dt)
    table = randn(device, (nb, H), 2, 0.7)
    lengths = starts = None
    if masks:
        lengths = torch.tensor([max(1, N - 7 * b - N // 3 * (b % 2)) for b in range(B)], device=device, dtype=torch.int32)
    if causal:
        starts = torch.tensor([max(0, (N if lengths is None else int(lengths[b])) - M) for b in range(B)], device=device, dtype=torch.int32)
    return x, table, lengths, starts, stx.rel_params(nb, dist, both, causal)


def rel_ref(x, table, mask, bucket, scale):
    """y and the largest |scale x| + |bias| of each row; rows without keys are zeros."""
    bias = table.to(F64)[bucket].permute(0, 3, 1, 2)
    z = (x.to(F64) * scale + bias).masked_fill(~mask[:, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top.isinf(), 0.0, top))
    s = e.sum(-1, keepdim=True)
    size = ((x.to(F64) * scale).abs() + bias.abs()).masked_fill(~mask[:, None], 0.0).amax(-1, keepdim=True)
    return torch.where(s > 0, e / s, 0.0), size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", REL, ids=lambda s: "-".join(str(v) for v in s))
def test_soft_max_rel(device, dtype, shape):
    B, H, M, N, nb, dist, both, causal, _ = shape
    x, table, lengths, starts, p = rel_inputs(device, TYPES[dtype], shape)
    mask, rel = seen_ref(B, M, N, lengths, starts, causal, device)
    want, size = rel_ref(x, table, mask, buckets_ref(rel, nb, dist, both), 0.25)
    x.masked_fill_(~mask[:, None], math.nan)                     # what is masked is not looked at
    got = stx.soft_max_rel(x, table, p, 0.25, lengths, starts)
    per_lane = N / 64 if N <= 1024 else N / 256 + 16
    close(got, want, want * (10 * size + 8 + 2 * (per_lane + 16)) * U, "y")
    assert bool((got[~mask[:, None].expand_as(got)] == 0).all())
    stx.soft_max_rel(x, table, p, 0.25, lengths, starts, out=x)
    assert torch.equal(x, got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", REL, ids=lambda s: "-".join(str(v) for v in s))
def test_soft_max_rel_back(device, dtype, shape):
    B, H, M, N, nb, dist, both, causal, _ = shape
    x, table, lengths, starts, p = rel_inputs(device, TYPES[dtype], shape)
    mask, rel = seen_ref(B, M, N, lengths, starts, causal, device)
    bucket = buckets_ref(rel, nb, dist, both)
    y = rel_ref(x, table, mask, bucket, 0.25)[0].to(x.dtype)
    dy = randn(device, x.shape, 3, dtype=x.dtype)
    g = y.to(F64) * (dy.to(F64) - (y.to(F64) * dy.to(F64)).sum(-1, keepdim=True))
    dtable = torch.zeros(nb, H, dtype=F64, device=device)
    size = torch.zeros_like(dtable)
    for k in range(nb):
        here = (bucket == k)[:, None]
        dtable[k], size[k] = (torch.where(here, v, 0.0).sum((0, 2, 3)) for v in (g, g.abs()))
    for t in (y, dy):
        t.masked_fill_(~mask[:, None], math.nan)
    dx, dt = stx.soft_max_rel_back(dy, y, p, 0.25, lengths, starts)
    close(dx, g * 0.25, 2 * U * (g * 0.25).abs(), "dx")
    close(dt, dtable, 2.0 ** -45 * size, "dtable")
    again = stx.soft_max_rel_back(dy, y, p, 0.25, lengths, starts)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dt)
    assert torch.equal(stx.soft_max_rel_back(dy, y, p, 0.25, lengths, starts, dtable=False)[0], dx)


@pytest.mark.parametrize("nb,dist,both", [(32, 128, True), (32, 128, False), (256, 2048, True), (256, 2048, False), (8, 27, False), (4, 2, True), (2, 2, False),
                                          (16, 81, False), (128, 33, True)])
def test_rel_buckets(device, nb, dist, both):
    """Every distance's bucket, borders that are whole numbers among them: a table that lets one bucket a head through."""
    N = 2 * dist + 9
    table = torch.full((nb, nb), -math.inf, device=device)
    table.fill_diagonal_(0.0)
    x = torch.zeros((1, nb, 1, N), device=device)
    start = torch.tensor([N // 2], dtype=torch.int32, device=device)
    y = stx.soft_max_rel(x, table, stx.rel_params(nb, dist, both), starts=start)
    want = buckets_ref(torch.arange(N, device=device) - N // 2, nb, dist, both)
    assert torch.equal(y[0, :, 0] > 0, want == torch.arange(nb, device=device)[:, None])


@pytest.mark.parametrize("causal", [False, True])
def test_rel_masks_at_their_limits(device, causal):
    """Lengths of zero, below zero and past the keys; starts far before, past the keys and at the type's limits."""
    lengths = torch.tensor([0, -5, 1, 40, 1000, 2 ** 31 - 1, -2 ** 31, 17], dtype=torch.int32, device=device)
    starts = torch.tensor([0, 3, -1, -9, 100, 2 ** 31 - 1, -2 ** 31, -2 ** 31], dtype=torch.int32, device=device)
    B, H, M, N = 8, 2, 12, 40
    x, table = randn(device, (B, H, M, N), 1), randn(device, (32, H), 2)
    p = stx.rel_params(causal=causal)
    mask, rel = seen_ref(B, M, N, lengths, starts, causal, device)
    want, size = rel_ref(x, table, mask, buckets_ref(rel, 32, 128, True), 1.0)
    got = stx.soft_max_rel(x, table, p, 1.0, lengths, starts)
    close(got, want, want * (10 * size + 50) * U, "y")
    dy = randn(device, x.shape, 3)
    dx, dt = stx.soft_max_rel_back(dy, got, p, 1.0, lengths, starts)
    assert bool((dx[~mask[:, None].expand_as(dx)] == 0).all()) and bool(dt.isfinite().all())


def test_rel_infinite_scores(device):
    """Scores of -infinity are keys left out; a row of them alone is zeros; the type's lowest value is a score as any."""
    x = torch.zeros((1, 1, 4, 70), device=device)
    x[0, 0, 0, 5:] = -math.inf
    x[0, 0, 1] = -math.inf
    x[0, 0, 2] = torch.finfo(torch.float32).min
    x[0, 0, 3, 0] = math.nan
    table = torch.zeros((32, 1), device=device)
    y = stx.soft_max_rel(x, table, stx.rel_params(), 0.25)
    assert torch.allclose(y[0, 0, 0, :5], torch.full((5,), 0.2, device=device)) and bool((y[0, 0, 0, 5:] == 0).all())
    assert bool((y[0, 0, 1] == 0).all()) and torch.allclose(y[0, 0, 2], torch.full((70,), 1 / 70, device=device))
    assert bool(y[0, 0, 3].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [3, 70, 700, 5000, 20000])
def test_rel_lowest_values(device, dtype, N):
    """Keys hidden by the type's lowest value, at scale 1, in rows of every width: none of the sum beside other
    scores, an equal share each where a row has nothing else, and so beside -infinity; and biases of the lowest float.
    Exponentials and their sums are exact here; 8 u are the quotient's."""
    dt = TYPES[dtype]
    low = torch.finfo(dt).min
    x = torch.zeros((1, 1, 5, N), dtype=dt, device=device)
    x[0, 0, 0, 2:] = low
    x[0, 0, 1] = low
    x[0, 0, 2] = -math.inf
    x[0, 0, 2, N - 2:] = low
    x[0, 0, 3, 1:] = torch.finfo(dt).max
    x[0, 0, 4, 0] = low
    y = stx.soft_max_rel(x, torch.zeros((32, 1), device=device), stx.rel_params(), 1.0)
    wide = x[0, 0].to(F64)
    want = torch.softmax(wide, -1)
    close(y[0, 0], want, 8 * U * want, "y")
    table = torch.full((32, 1), torch.finfo(torch.float32).min, device=device)
    y = stx.soft_max_rel(torch.zeros_like(x), table, stx.rel_params(), 1.0)
    want = torch.full_like(want, 1 / N)
    close(y[0, 0], want, 8 * U * want, "y")


def test_rel_strides_and_empty(device):
    """Rows of a wider buffer at odd offsets, its other elements as they were; calls of no elements."""
    B, H, M, N = 2, 3, 33, 45
    p = stx.rel_params(16, 30)
    table = randn(device, (16, H), 2)
    for dt in TYPES.values():
        wide = randn(device, (H, B, M, N + 5), 1, dtype=dt)
        x = wide.transpose(0, 1)[..., 3:3 + N]
        want = stx.soft_max_rel(x.contiguous(), table, p)
        out = torch.full((B, H, M + 1, N + 3), 7.0, device=device, dtype=dt)
        stx.soft_max_rel(x, table, p, out=out[:, :, 1:, 1:1 + N])
        assert torch.equal(out[:, :, 1:, 1:1 + N], want)
        out[:, :, 1:, 1:1 + N] = 7.0
        assert bool((out == 7.0).all())
        dwide = randn(device, (B, H, M, N + 1), 4, dtype=dt)
        dx, dt_ = stx.soft_max_rel_back(dwide[..., 1:], want, p)
        dx2, dt2 = stx.soft_max_rel_back(dwide[..., 1:].contiguous(), want, p)
        assert torch.equal(dx, dx2) and torch.equal(dt_, dt2)
    for shape in ((0, H, M, N), (B, H, 0, N), (B, H, M, 0)):
        x = torch.empty(shape, device=device)
        assert stx.soft_max_rel(x, table, p).shape == x.shape
        dx, dt_ = stx.soft_max_rel_back(x, x, p)
        assert dx.shape == x.shape and torch.equal(dt_, torch.zeros(16, H, device=device))


def test_rel_gradient_against_differences(device):
    B, H, M, N = 1, 2, 5, 9
    x, table, dy = randn(device, (B, H, M, N), 1), randn(device, (8, H), 2), randn(device, (B, H, M, N), 3)
    p = stx.rel_params(8, 6, True, True)
    starts = torch.tensor([3], dtype=torch.int32, device=device)
    mask, rel = seen_ref(B, M, N, None, starts, True, device)
    bucket = buckets_ref(rel, 8, 6, True)
    dx, dt = stx.soft_max_rel_back(dy, stx.soft_max_rel(x, table, p, 0.5, None, starts), p, 0.5, None, starts)
    f = lambda x, w: float((rel_ref(x, w, mask, bucket, 0.5)[0] * dy.to(F64)).sum())  # noqa: E731
    step = 1e-5
    for t, got in ((x, dx), (table, dt)):
        for i in range(0, t.numel(), 3):
            d = torch.zeros_like(t, dtype=F64).view(-1)
            d[i] = step
            d, t64 = d.view_as(t), t.to(F64)
            diff = (f(t64 + d, table) - f(t64 - d, table) if t is x else f(x, t64 + d) - f(x, t64 - d)) / (2 * step)
            assert abs(float(got.reshape(-1)[i]) - diff) < 1e-5 * max(1.0, abs(diff))


# ------------------------------------------------------------------------ differential attention
DIFF = [
    # B, M, N, H, Hk, D, V, causal, masks
    (1, 1, 1, 1, 1, 64, 128, False, None),
    (2, 1, 300, 8, 2, 64, 128, True, "ragged"),               # single tokens: waves and blocks split the keys
    (3, 1, 5000, 4, 4, 64, 128, True, "ragged"),
    (2, 3, 700, 8, 2, 128, 256, True, "ragged"),
    (1, 16, 1000, 1, 1, 128, 128, False, None),
    (2, 4, 400, 4, 1, 32, 64, False, "ragged"),
    (1, 2, 130, 2, 1, 64, 64, True, None),
    (2, 60, 60, 4, 4, 64, 128, False, None),
    (1, 801, 801, 4, 4, 64, 128, False, "ragged"),
    (2, 131, 260, 8, 2, 64, 128, True, "ragged"),
    (1, 200, 200, 4, 2, 64, 64, True, None),
    (1, 129, 333, 4, 2, 128, 256, True, "ragged"),
    (1, 70, 190, 2, 2, 96, 96, False, None),                   # rows padded in LDS
    (1, 150, 150, 6, 2, 40, 80, True, None),
    (2, 90, 77, 3, 3, 32, 32, True, None),                     # more queries than keys
    (1, 65, 100, 2, 1, 33, 47, True, "ragged"),                # rows that are not whole chunks
    (1, 9, 50, 2, 1, 1, 1, False, None),
]


def diff_inputs(device, dt, shape, pad=None):
    B, M, N, H, Hk, D, V, causal, masks = shape
    q, k, v = (randn(device, s, 1 + i, dtype=dt) for i, s in enumerate(((B, M, 2 * H, D), (B, N, 2 * Hk, D), (B, N, Hk, V))))
    lam = randn(device, (H,), 4, 0.2, 0.5)
    lengths = starts = None
    if masks:
        lengths = torch.tensor([max(1, N - 7 * b - N // 3 * (b % 2)) for b in range(B)], device=device, dtype=torch.int32)
    if causal:
        starts = torch.tensor([max(0, (N if lengths is None else int(lengths[b])) - M) for b in range(B)], device=device, dtype=torch.int32)
    return q, k, v, lam, lengths, starts


def diff_maps(q, k, v, mask, scale):
    """Both maps P (2, B, H, M, N), ln sum exp (B, H, 2, M), Z and the operands repeated for each head, in 64 bits."""
    B, M, H2, D = q.shape
    H, Hk = H2 // 2, v.shape[2]
    q = q.to(F64).view(B, M, H, 2, D).permute(3, 0, 2, 1, 4).contiguous()
    k = k.to(F64).view(B, -1, Hk, 2, D).permute(3, 0, 2, 1, 4).repeat_interleave(H // Hk, 2).contiguous()
    v = v.to(F64).permute(0, 2, 1, 3).repeat_interleave(H // Hk, 1).contiguous()
    kt = k.transpose(3, 4).contiguous()
    z = (torch.matmul(q, kt) * scale).masked_fill(~mask[:, None], -math.inf)
    size = (torch.matmul(q.abs(), kt.abs()) * scale).masked_fill(~mask[:, None], 0.0).amax(-1, keepdim=True)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), 0.0, top)
    e = torch.exp(z - top)
    s = e.sum(-1, keepdim=True)
    lse = (top + torch.log(s)).squeeze(-1).permute(1, 2, 0, 3)
    return torch.where(s > 0, e / s, 0.0), lse, size, q, k, v


def spoil(k, v, lengths):
    """Keys from a sequence's length on hold NaN."""
    if lengths is not None:
        for b, n in enumerate(lengths.tolist()):
            k[b, n:] = math.nan
            v[b, n:] = math.nan


def check_diff(got, q, k, v, lam, mask, scale, what, norms=True):
    out, second, lse = got
    p, want_lse, size, _, _, v64 = diff_maps(q, k, v, mask, scale)
    D, N = q.shape[3], k.shape[1]
    o = [torch.matmul(m, v64) for m in p]
    h = half_step(q.dtype) if q.dtype != torch.float32 else 0.0
    off = [(2 * (D + 8) * U * size[m] + h + (8 + 4 * math.sqrt(N)) * U) * torch.matmul(p[m], v64.abs()) for m in range(2)]
    lam = lam.to(F64)[:, None, None]
    want = (o[0] - lam * o[1]).transpose(1, 2)
    close(out, want, (off[0] + lam.abs() * off[1]).transpose(1, 2), what + " out")
    if norms and N >= 64:
        norm_close(out, want, 2, what + " out")
    if second is not None:
        close(second, o[1].transpose(1, 2), off[1].transpose(1, 2), what + " second")
        seen = want_lse > -math.inf
        assert bool((lse[~seen] == -math.inf).all())
        bound = ((D + 8) * U * size.squeeze(-1).permute(1, 2, 0, 3) + (16 + math.sqrt(N)) * U) + 4 * U * want_lse.abs()
        assert bool(((lse.to(F64) - want_lse).abs() <= bound)[seen].all()), what + " lse"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", DIFF, ids=lambda s: "-".join(str(v) for v in s))
def test_diff_attention(device, dtype, shape):
    B, M, N, H, Hk, D, V, causal, _ = shape
    q, k, v, lam, lengths, starts = diff_inputs(device, TYPES[dtype], shape)
    mask, _ = seen_ref(B, M, N, lengths, starts, causal, device)
    kept, v_kept = k.clone(), v.clone()
    spoil(k, v, lengths)
    got = stx.diff_attention(q, k, v, lam, causal=causal, lengths=lengths, starts=starts, keep=True)
    check_diff(got, q, kept, v_kept, lam, mask, D ** -0.5, "diff")
    alone = stx.diff_attention(q, k, v, lam, causal=causal, lengths=lengths, starts=starts)
    assert torch.equal(alone[0], got[0]) and alone[1] is None and alone[2] is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 20, 70])
@pytest.mark.parametrize("causal", [False, True])
def test_diff_masks_at_their_limits(device, dtype, M, causal):
    """Rows that see no key; lengths and starts at and past their limits."""
    lengths = torch.tensor([0, -5, 1, 40, 1000, 2 ** 31 - 1, -2 ** 31, 17], dtype=torch.int32, device=device)
    starts = torch.tensor([0, 3, -1, -9, 100, 2 ** 31 - 1, -2 ** 31, -2 ** 31], dtype=torch.int32, device=device)
    B, N, H, Hk, D, V = 8, 90, 4, 2, 64, 128
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (B, M, N, H, Hk, D, V, False, None))
    mask, _ = seen_ref(B, M, N, lengths, starts, causal, device)
    got = stx.diff_attention(q, k, v, lam, causal=causal, lengths=lengths, starts=starts, keep=True)
    check_diff(got, q, k, v, lam, mask, D ** -0.5, "limits", norms=False)
    nothing = ~mask.any(-1)
    for t in got[:2]:
        assert bool((t[nothing] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_diff_strides_and_neighbours(device, dtype):
    """q, k and v as slices of projections, at unaligned offsets too, a cache longer than its keys, outputs into wider
    buffers whose other elements stay."""
    B, M, N, H, Hk, D, V = 2, 37, 90, 4, 2, 64, 128
    dt = TYPES[dtype]
    for shift in (0, 3):
        wide = randn(device, (B, M, 2 * H * D + 13), 1, dtype=dt)
        q = wide[..., shift:shift + 2 * H * D].unflatten(-1, (2 * H, D))
        cache = randn(device, (B, N + 30, Hk, 2 * D + V + 16), 2, dtype=dt)
        k = cache[:, 5:5 + N, :, shift:shift + 2 * D]
        k = k.reshape(B, N, 2 * Hk, D)
        v = cache[:, 5:5 + N, :, 2 * D + shift:2 * D + shift + V]
        lam = randn(device, (H,), 4, 0.2, 0.5)
        mask, _ = seen_ref(B, M, N, None, None, False, device)
        want = stx.diff_attention(q.contiguous(), k.contiguous(), v.contiguous(), lam, keep=True)
        buffers = [torch.full((B, M + 2, H, V + 5), 7.0, device=device, dtype=dt) for _ in range(2)]
        out, second = (t[:, 1:M + 1, :, shift:shift + V] for t in buffers)
        got = stx.diff_attention(q, k, v, lam, keep=True, out=out, second=second)
        if shift == 0:
            assert torch.equal(out, want[0]) and torch.equal(second, want[1]) and torch.equal(got[2], want[2])
        check_diff(got, q, k, v, lam, mask, D ** -0.5, "strides")
        for t, s in zip(buffers, (out, second)):
            s.fill_(7.0)
            assert bool((t == 7.0).all())


def test_diff_empty(device):
    lam = torch.ones(2, device=device)
    make = lambda B, M, N: (torch.empty(B, M, 4, 8, device=device), torch.empty(B, N, 2, 8, device=device), torch.empty(B, N, 1, 8, device=device))  # noqa: E731
    for B, M, N in ((0, 3, 3), (2, 0, 3)):
        assert stx.diff_attention(*make(B, M, N), lam, keep=True)[0].shape == (B, M, 2, 8)
    out, second, lse = stx.diff_attention(*make(2, 3, 0), lam, keep=True)
    assert bool((out == 0).all()) and bool((second == 0).all()) and bool((lse == -math.inf).all())


def diff_back_ref(dy, q, k, v, lam, out, second, lse, mask, scale):
    """(gradient, bound of its error before rounding) of each, from what the forward call kept, in 64 bits. With E = (2 (D + 8) Z
    + 8 |lse| + 16) u relative to P, dP off by (V + 8) u Y (Y = |dy| |v|^T) and D by (V + 8) u sum |dy| (|out| + 2 |lam
    second|), dS = f P (dP - D) is off by |f| (E P |dP - D| + P (both)) and, rounded, by h |dS| more; sums drift by 4 sqrt(n) u."""
    B, M, H2, D = q.shape
    H, Hk, V, N = H2 // 2, v.shape[2], v.shape[3], k.shape[1]
    g = H // Hk
    h = half_step(q.dtype) if q.dtype != torch.float32 else 0.0
    p, _, size, q64, k64, v64 = diff_maps(q, k, v, mask, scale)
    z = torch.matmul(q64, k64.transpose(3, 4).contiguous()) * scale
    ls = lse.to(F64).permute(2, 0, 1, 3)[..., None]
    p = torch.where(mask[:, None], torch.exp(z - ls), 0.0)
    E = (2 * (D + 8) * size + 8 * torch.where(ls.isinf(), 0.0, ls.abs()) + 16) * U
    y, o, o2 = (t.to(F64).transpose(1, 2).contiguous() for t in (dy, out, second))
    la = lam.to(F64)[:, None, None]
    vt = v64.transpose(2, 3).contiguous()
    dp, Y = torch.matmul(y, vt), torch.matmul(y.abs(), vt.abs())
    dots = ((y * (o + la * o2)).sum(-1, keepdim=True), (y * o2).sum(-1, keepdim=True))
    ddot = (V + 8) * U * (y.abs() * (o.abs() + 2 * (la * o2).abs())).sum(-1, keepdim=True)
    dq, bq = (torch.zeros(2, B, H, M, D, dtype=F64, device=q.device) for _ in range(2))
    dk, bk = (torch.zeros(2, B, H, N, D, dtype=F64, device=q.device) for _ in range(2))
    tiny = 2.0 ** -38 * V * float(v64[~v64.isnan()].abs().max()) * float(y.abs().max()) * max(1.0, float(la.abs().max())) if q.dtype == torch.float16 else 0.0
    for m, f in ((0, torch.ones_like(la)), (1, -la)):
        ds = f * p[m] * (dp - dots[m])
        e = f.abs() * p[m] * (E[m] * (dp - dots[m]).abs() + (V + 8) * U * Y + ddot) + h * ds.abs() + tiny * mask[:, None]
        dq[m], dk[m] = torch.matmul(ds, k64[m]) * scale, torch.matmul(ds.transpose(2, 3).contiguous(), q64[m]) * scale
        bq[m] = torch.matmul(e + 4 * math.sqrt(N) * U * ds.abs(), k64[m].abs()) * scale
        bk[m] = torch.matmul((e + 4 * math.sqrt(M * g) * U * ds.abs()).transpose(2, 3).contiguous(), q64[m].abs()) * scale
    mix = (p[0] - la * p[1]).transpose(2, 3).contiguous()
    both = (p[0] * (E[0] + h + 4 * math.sqrt(M * g) * U) + la.abs() * p[1] * (E[1] + h + 4 * math.sqrt(M * g) * U)).transpose(2, 3).contiguous()
    dv, bv = torch.matmul(mix, y), torch.matmul(both, y.abs())
    dlam = -(p[1] * dp).sum((0, 2, 3))
    bl = (p[1] * (E[1] * dp.abs() + (V + 8) * U * Y) + (math.sqrt(N) + 16) * U * (p[1] * dp).abs()).sum((0, 2, 3))
    heads = lambda t: t.unflatten(1, (Hk, g)).sum(2)  # noqa: E731
    rows = lambda t: t.permute(1, 3, 2, 0, 4).reshape(B, M, 2 * H, D)  # noqa: E731
    keys = lambda t: torch.stack([heads(x) for x in t]).permute(1, 3, 2, 0, 4).reshape(B, N, 2 * Hk, D)  # noqa: E731
    return (rows(dq), rows(bq)), (keys(dk), keys(bk)), (heads(dv).transpose(1, 2), heads(bv).transpose(1, 2)), (dlam, bl)


def check_diff_back(got, dy, q, k, v, lam, kept, mask, scale, what, norms=True):
    want = diff_back_ref(dy, q, k, v, lam, *kept, mask, scale)
    for g, (w, bound), name in zip(got, want, ("dq", "dk", "dv", "dlam")):
        close(g, w, bound, f"{what} {name}")
        if norms and name != "dlam" and min(q.shape[1], k.shape[1]) >= 64:
            norm_close(g, w, 2, f"{what} {name}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", DIFF, ids=lambda s: "-".join(str(v) for v in s))
def test_diff_attention_back(device, dtype, shape):
    B, M, N, H, Hk, D, V, causal, _ = shape
    q, k, v, lam, lengths, starts = diff_inputs(device, TYPES[dtype], shape)
    dy = randn(device, (B, M, H, V), 7, dtype=q.dtype)
    mask, _ = seen_ref(B, M, N, lengths, starts, causal, device)
    kc, vc = k.clone(), v.clone()
    spoil(k, v, lengths)
    masks = dict(causal=causal, lengths=lengths, starts=starts)
    kept = stx.diff_attention(q, k, v, lam, keep=True, **masks)
    got = stx.diff_attention_back(dy, q, k, v, lam, *kept, **masks)
    check_diff_back(got, dy, q, kc, vc, lam, kept, mask, D ** -0.5, "back")
    if lengths is not None:
        for b, n in enumerate(lengths.tolist()):
            assert bool((got[1][b, n:] == 0).all()) and bool((got[2][b, n:] == 0).all())
    again = stx.diff_attention_back(dy, q, k, v, lam, *kept, **masks)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 70])
@pytest.mark.parametrize("causal", [False, True])
def test_diff_back_masks_at_their_limits(device, dtype, M, causal):
    lengths = torch.tensor([0, -5, 1, 40, 1000, 2 ** 31 - 1, -2 ** 31, 17], dtype=torch.int32, device=device)
    starts = torch.tensor([0, 3, -1, -9, 100, 2 ** 31 - 1, -2 ** 31, -2 ** 31], dtype=torch.int32, device=device)
    B, N, H, Hk, D, V = 8, 90, 4, 2, 64, 128
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (B, M, N, H, Hk, D, V, False, None))
    dy = randn(device, (B, M, H, V), 7, dtype=q.dtype)
    mask, _ = seen_ref(B, M, N, lengths, starts, causal, device)
    masks = dict(causal=causal, lengths=lengths, starts=starts)
    kept = stx.diff_attention(q, k, v, lam, keep=True, **masks)
    got = stx.diff_attention_back(dy, q, k, v, lam, *kept, **masks)
    check_diff_back(got, dy, q, k, v, lam, kept, mask, D ** -0.5, "limits", norms=False)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1e-6, 1.0, 3e3])
def test_diff_back_range(device, dtype, size):
    """Gradients far from 1, and rows whose gradient is a small part of the largest: fp16 keeps its bits."""
    B, M, N, H, Hk, D, V = 1, 80, 150, 2, 1, 64, 128
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (B, M, N, H, Hk, D, V, False, None))
    dy = (randn(device, (B, M, H, V), 7) * (size if size > 1e-3 else 1e-2))
    dy[:, ::3] *= 1e-2
    dy, mask = dy.to(q.dtype), torch.ones(B, M, N, dtype=torch.bool, device=device)
    kept = stx.diff_attention(q, k, v, lam, keep=True)
    got = stx.diff_attention_back(dy, q, k, v, lam, *kept)
    check_diff_back(got, dy, q, k, v, lam, kept, mask, D ** -0.5, "range", norms=size >= 1.0)


def test_diff_gradient_against_differences(device):
    """The whole way, forward and backward in fp32, against central differences of the definition in 64 bits."""
    B, M, N, H, Hk, D, V = 1, 5, 7, 2, 1, 16, 16
    q, k, v, lam, _, _ = diff_inputs(device, torch.float32, (B, M, N, H, Hk, D, V, False, None))
    starts = torch.tensor([2], dtype=torch.int32, device=device)
    mask, _ = seen_ref(B, M, N, None, starts, True, device)
    dy = randn(device, (B, M, H, V), 7)
    kept = stx.diff_attention(q, k, v, lam, causal=True, starts=starts, keep=True)
    grads = stx.diff_attention_back(dy, q, k, v, lam, *kept, causal=True, starts=starts)

    def f(q, k, v, lam):
        p, _, _, _, _, v64 = diff_maps(q, k, v, mask, D ** -0.5)
        o = torch.matmul(p[0], v64) - lam.to(F64)[:, None, None] * torch.matmul(p[1], v64)
        return float((o.transpose(1, 2) * dy.to(F64)).sum())

    args = [t.to(F64) for t in (q, k, v, lam)]
    step = 1e-5
    for a, grad in enumerate(grads):
        for i in range(0, args[a].numel(), 5 if args[a].numel() > 2 else 1):
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in args]
                moved[a].view(-1)[i] += sign * step
                ends.append(f(*moved))
            diff = (ends[0] - ends[1]) / (2 * step)
            assert abs(float(grad.reshape(-1)[i]) - diff) < 2e-5 * max(1.0, abs(diff)), (a, i)


def test_diff_back_strides_and_empty(device):
    """Gradients into slices of wider buffers, from operands at unaligned offsets; calls without queries or keys."""
    B, M, N, H, Hk, D, V = 2, 37, 90, 4, 2, 64, 128
    for dt in TYPES.values():
        q, k, v, lam, _, _ = diff_inputs(device, dt, (B, M, N, H, Hk, D, V, False, None))
        dy = randn(device, (B, M, H, V), 7, dtype=dt)
        kept = stx.diff_attention(q, k, v, lam, keep=True)
        mask = torch.ones(B, M, N, dtype=torch.bool, device=device)
        shifted = []
        for t in (q, k, v, dy):
            w = torch.zeros((*t.shape[:2], t.shape[2] + 1, t.shape[3] + 3), device=device, dtype=dt)
            w[:, :, 1:, 3:] = t
            shifted.append(w[:, :, 1:, 3:])
        outs = [torch.full((t.shape[0], t.shape[1] + 1, t.shape[2], t.shape[3] + 5), 7.0, device=device, dtype=dt) for t in (q, k, v)]
        into = [t[:, 1:, :, 2:2 + n] for t, n in zip(outs, (D, D, V))]
        got = stx.diff_attention_back(shifted[3], *shifted[:3], lam, *kept, dq=into[0], dk=into[1], dv=into[2])
        check_diff_back(got, dy, q, k, v, lam, kept, mask, D ** -0.5, "strides")
        for t, s in zip(outs, into):
            s.fill_(7.0)
            assert bool((t == 7.0).all())
    lam = torch.ones(2, device=device)
    for b, m, n in ((0, 3, 3), (2, 0, 3), (2, 3, 0)):
        q, k, v = torch.ones(b, m, 4, 8, device=device), torch.ones(b, n, 2, 8, device=device), torch.ones(b, n, 1, 8, device=device)
        kept = stx.diff_attention(q, k, v, lam, keep=True)
        got = stx.diff_attention_back(torch.ones(b, m, 2, 8, device=device), q, k, v, lam, *kept)
        assert all(bool((t == 0).all()) for t in got) and got[3].shape == (2,)


# ----------------------------------------------------------------------- together, graphs, streams
def attention_layer(x, w, pos, rope, lam, p, table, masks, keep):
    """Differential attention over normed and rotated q and k, plus a pass of ordinary attention with a position bias."""
    B, N, D = x.shape
    H, dh = 4, 32
    qkv = (x @ w.t()).view(B, N, 3 * H, dh)
    q, k = stx.qk_norm_rope(qkv[:, :, :H], pos, rope, p["wq"], qkv[:, :, H:2 * H], p["wk"])
    v = qkv[:, :, 2 * H:].reshape(B, N, H // 2, 2 * dh)
    out, second, lse = stx.diff_attention(q, k, v, lam, keep=True, **masks)
    score = torch.matmul(q.transpose(1, 2).float().contiguous(), k.permute(0, 2, 3, 1).float().contiguous()).to(x.dtype)
    y = stx.soft_max_rel(score, table, p["rel"], dh ** -0.5, masks["lengths"], masks["starts"])
    keep.update(qkv=qkv, q=q, k=k, v=v, out=out, second=second, lse=lse, y=y)
    return out, y


def layer_inputs(device, dt, seed=0):
    B, N, D, H, dh = 2, 77, 96, 4, 32
    r = lambda *s, seed, scale=1.0, t=dt: randn(device, s, seed, scale, dtype=t)  # noqa: E731
    x, w = r(B, N, D, seed=seed + 1), r(3 * H * dh, D, seed=2, scale=D ** -0.5)
    p = {"wq": r(H, dh, seed=3, scale=0.3, t=torch.float32) + 1, "wk": r(H, dh, seed=4, scale=0.3, t=torch.float32) + 1,
         "rel": stx.rel_params(16, 40, False, True)}
    lam, table = r(H // 2, seed=5, scale=0.2, t=torch.float32) + 0.5, r(16, H, seed=6, t=torch.float32)
    masks = dict(causal=True, lengths=torch.tensor([N, N - 20], dtype=torch.int32, device=device), starts=torch.zeros(2, dtype=torch.int32, device=device))
    return x, w, torch.arange(N, device=device, dtype=torch.int32), stx.rope_params(dh, 2), lam, p, table, masks


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_together(device, dtype):
    """The operators one after another, forward and backward, against the layer in 64 bits and its gradients by autograd. The
    roundings of qkv, q and k, the maps and the results (and of their gradients on the way back) lie one after another, each
    relative to values that pass on with a gain of about 1 (scores: of their size, 6 at most here, so 6 h each): 24 h in
    the 2-norm forward, twice that backward."""
    dt = TYPES[dtype]
    x, w, pos, rope, lam, p, table, masks = layer_inputs(device, dt)
    B, N, D = x.shape
    H, dh = 4, 32
    kept = {}
    out, y = attention_layer(x, w, pos, rope, lam, p, table, masks, kept)
    dout, dy = randn(device, out.shape, 11, dtype=dt), randn(device, y.shape, 12, dtype=dt)
    dq, dk, dv, dlam = stx.diff_attention_back(dout, kept["q"], kept["k"], kept["v"], lam, out, kept["second"], kept["lse"], **masks)
    dscore, dtable = stx.soft_max_rel_back(dy, y, p["rel"], dh ** -0.5, masks["lengths"], masks["starts"])
    dq = dq + torch.matmul(dscore.float(), kept["k"].transpose(1, 2).float().contiguous()).transpose(1, 2).to(dt)
    dk = dk + torch.matmul(dscore.transpose(2, 3).float().contiguous(), kept["q"].transpose(1, 2).float().contiguous()).transpose(1, 2).to(dt)
    qkv = kept["qkv"]
    dqp, dwq, dkp, dwk = stx.qk_norm_rope_back(dq, qkv[:, :, :H], pos, rope, p["wq"], dk, qkv[:, :, H:2 * H], p["wk"])
    dqkv = torch.cat([dqp, dkp, dv.reshape(B, N, H, dh)], 2).view(B, N, -1)
    got = {"out": out, "y": y, "dx": dqkv @ w, "dlam": dlam, "dtable": dtable, "dwq": dwq, "dwk": dwk}

    # in 64 bits, on the CPU (batched products of transposed views)
    leaf = lambda t: t.to(F64).cpu().requires_grad_()  # noqa: E731
    x6, wq6, wk6, lam6, table6 = (leaf(t) for t in (x, p["wq"], p["wk"], lam, table))
    qkv6 = (x6 @ w.to(F64).cpu().t()).view(B, N, 3 * H, dh)
    theta = pos.to(F64).cpu()[:, None, None] * 10000.0 ** (-2.0 * torch.arange(dh // 2, dtype=F64) / dh)

    def turned(t, wt):
        z = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * wt
        a, b = z[..., :dh // 2], z[..., dh // 2:]
        return torch.cat([a * theta.cos() - b * theta.sin(), a * theta.sin() + b * theta.cos()], -1)

    q6, k6 = turned(qkv6[:, :, :H], wq6), turned(qkv6[:, :, H:2 * H], wk6)
    v6 = qkv6[:, :, 2 * H:].reshape(B, N, H // 2, 2 * dh)
    mask, rel = (t.cpu() for t in seen_ref(B, N, N, masks["lengths"], masks["starts"], True, device))
    z = torch.einsum("bihd,bjhd->bhij", q6, k6) * dh ** -0.5
    maps = torch.softmax(z.masked_fill(~mask[:, None], -math.inf), -1)
    out6 = torch.einsum("bhij,bjhd->bihd", maps[:, 0::2] - lam6[:, None, None] * maps[:, 1::2], v6)
    y6 = torch.softmax((z + table6[buckets_ref(rel, 16, 40, False)].permute(0, 3, 1, 2)).masked_fill(~mask[:, None], -math.inf), -1)
    ((out6 * dout.to(F64).cpu()).sum() + (y6 * dy.to(F64).cpu()).sum()).backward()
    want = {"out": out6, "y": y6, "dx": x6.grad, "dlam": lam6.grad, "dtable": table6.grad, "dwq": wq6.grad, "dwk": wk6.grad}
    h = half_step(dt)
    for name, t in got.items():
        ref = want[name].detach()
        off = float((t.to(F64).cpu() - ref).norm() / ref.norm())
        assert off <= (24 if name in ("out", "y") else 48) * h, (name, off)


def test_graph_replays_and_streams(device):
    """A captured forward and backward run of the operators, single tokens and split keys among it, replayed on new data with
    eager calls between, on a stream of its own: the eager results each time."""
    dt = torch.float16                                          # with the kernels that only fp16 has
    x, w, pos, rope, lam, p, table, masks = layer_inputs(device, dt)
    dout = randn(device, (2, 77, 2, 64), 21, dtype=dt)
    token, cache_k, cache_v = (randn(device, s, 22 + i, dtype=dt) for i, s in enumerate(((2, 1, 4, 32), (2, 3000, 4, 32), (2, 3000, 2, 64))))

    def step(s=None):
        qkv = x @ w.t()
        qkv = qkv.view(2, 77, 12, 32)
        q, k = stx.qk_norm_rope(qkv[:, :, :4], pos, rope, p["wq"], qkv[:, :, 4:8], p["wk"], stream=s)
        v = qkv[:, :, 8:].reshape(2, 77, 2, 64)
        kept = stx.diff_attention(q, k, v, lam, keep=True, stream=s, **masks)
        g = stx.diff_attention_back(dout, q, k, v, lam, *kept, stream=s, **masks)
        n = stx.qk_norm_rope_back(g[0], qkv[:, :, :4], pos, rope, p["wq"], g[1], qkv[:, :, 4:8], p["wk"], stream=s)
        score = qkv.view(2, 4, 77, 96)[..., :77]
        y = stx.soft_max_rel(score, table, p["rel"], 0.2, masks["lengths"], masks["starts"], stream=s)
        d = stx.soft_max_rel_back(score, y, p["rel"], 0.2, masks["lengths"], masks["starts"], stream=s)
        t = stx.diff_attention(token, cache_k, cache_v, lam, stream=s)[0]
        return [*kept, *g, *n, y, *d, t]

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
        x.copy_(randn(device, x.shape, 100 + rep, 1.0 + rep, dtype=dt))
        dout.copy_(randn(device, dout.shape, 200 + rep, 10.0 ** (rep - 2), dtype=dt))
        cache_k.copy_(randn(device, cache_k.shape, 300 + rep, dtype=dt))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), rep


def test_two_streams_at_once(device):
    """Two calls of each operator side by side give what they give alone."""
    sets = []
    for seed in (0, 50):
        q, k, v, lam, _, _ = diff_inputs(device, torch.bfloat16, (2, 200, 600, 4, 2, 64, 128, False, None))
        q = q * (1 + seed / 50)
        x, table = randn(device, (2, 4, 150, 300), seed, dtype=torch.bfloat16), randn(device, (32, 4), seed + 1)
        sets.append((q, k, v, lam, x, table))

    def run(a, s=None):
        q, k, v, lam, x, table = a
        kept = stx.diff_attention(q, k, v, lam, keep=True, stream=s)
        g = stx.diff_attention_back(kept[0], q, k, v, lam, *kept, stream=s)
        y = stx.soft_max_rel(x, table, stx.rel_params(), stream=s)
        return [*kept, *g, y, *stx.soft_max_rel_back(x, y, stx.rel_params(), stream=s)]

    want = [run(a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = [run(a, s) for a, s in zip(sets, streams)]
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(w, g))


def test_offsets_past_32_bits(device):
    """The last sequence of a cache of more than 2^32 bytes, rows of q and scores that far apart, and outputs there."""
    B, N, Hk, D, V, H = 3, 1500, 2, 64, 128, 4
    dt = torch.bfloat16
    far = (1 << 31) + 64                                          # elements from a sequence to the next
    cache = torch.empty(2 * far + N * Hk * (2 * D + V), device=device, dtype=dt)
    k = torch.as_strided(cache, (B, N, 2 * Hk, D), (far, Hk * (2 * D + V), D, 1))
    v = torch.as_strided(cache, (B, N, Hk, V), (far, Hk * (2 * D + V), V, 1), 2 * Hk * D)
    kc, vc = randn(device, (B, N, 2 * Hk, D), 1, dtype=dt), randn(device, (B, N, Hk, V), 2, dtype=dt)
    k.copy_(kc)
    v.copy_(vc)
    lam = randn(device, (H,), 4, 0.2, 0.5)
    for M in (1, 90):
        q, dy = randn(device, (B, M, 2 * H, D), 3, dtype=dt), randn(device, (B, M, H, V), 5, dtype=dt)
        kept = stx.diff_attention(q, kc, vc, lam, keep=True)
        got = stx.diff_attention(q, k, v, lam, keep=True)
        assert all(torch.equal(a, b) for a, b in zip(got, kept))
        want = stx.diff_attention_back(dy, q, kc, vc, lam, *kept)
        assert all(torch.equal(a, b) for a, b in zip(stx.diff_attention_back(dy, q, k, v, lam, *kept), want))
    x = torch.as_strided(cache, (B, 1, 20, 300), (far, 0, 1000, 1))
    table, p = randn(device, (32, 1), 6), stx.rel_params()
    xc = randn(device, (B, 1, 20, 300), 7, dtype=dt)
    x.copy_(xc)
    want = stx.soft_max_rel(xc, table, p)
    back = stx.soft_max_rel_back(xc, want, p)
    assert torch.equal(stx.soft_max_rel(x, table, p, out=x), want) and torch.equal(x, want)
    assert all(torch.equal(a, b) for a, b in zip(stx.soft_max_rel_back(xc, x, p), back))
    t = torch.as_strided(cache, (B, 20, 2, 64), (far, 128, 64, 1))
    tc = randn(device, (B, 20, 2, 64), 8, dtype=dt)
    t.copy_(tc)
    pos, r, w = torch.arange(20, device=device, dtype=torch.int32), stx.rope_params(64), torch.ones(64, device=device)
    want = stx.qk_norm_rope(tc, pos, r, w)
    assert torch.equal(stx.qk_norm_rope_back(tc, t, pos, r, w)[0], stx.qk_norm_rope_back(tc, tc, pos, r, w)[0])
    stx.qk_norm_rope(t, pos, r, w, out=t)
    assert torch.equal(t, want)


def test_outputs_belong_to_the_given_stream(device):
    """What a call allocates is on the stream that it runs on, the caller's being another."""
    s = torch.cuda.Stream()
    q, k, v, lam, _, _ = diff_inputs(device, torch.float32, (1, 3, 5, 2, 1, 16, 16, False, None))
    s.wait_stream(torch.cuda.current_stream())
    out, second, lse = stx.diff_attention(q, k, v, lam, keep=True, stream=s)
    s.synchronize()
    check_diff((out, second, lse), q, k, v, lam, torch.ones(1, 3, 5, dtype=torch.bool, device=device), 0.25, "stream")
