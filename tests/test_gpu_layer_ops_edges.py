"""The transformer-layer operators where ordinary data does not take them: intermediate values beyond the
data type's range and precision, operands of one sign, means far from zero, tails, other streams,
very many slices, offsets past 32 bits. References and bounds as in test_gpu_layer_ops."""
import math

import pytest

import stx
from test_gpu_layer_ops import ACTS, F64, TYPES, U, act_ref, close, ff_ref, half_step, norm_ref, randn, rope_ref  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ---------------------------------------------------------------------- gated block, backward
def ff_back_bounds(x, wg, wv, act, dh):
    """Gradients in 64 bits, bounded by the products' roundings alone: dg and dv, known to half a step of 16 bits
    (2^-17), enter each sum with that and with their own error as ff_ref has it; products of two parts
    leave out the two low ones (2^-17 once more). Three of them: 3 * 2^-17, less than an eighth of bf16's half step."""
    ref = ff_ref(x, wg, wv, act, None, None, dh)
    X, G, V, D = (t.to(F64) for t in (x, wg, wv, dh))
    g, v = torch.mm(X, G.t().contiguous()), torch.mm(X, V.t().contiguous())
    a, d = act_ref(g, act)
    dg, dv = D * v * d, D * a
    K, N, M = x.shape[1], wg.shape[0], x.shape[0]
    walk = 4 * math.sqrt(K) * U
    eg, ev = walk * torch.mm(X.abs(), G.abs().t().contiguous()) + U * g.abs(), walk * torch.mm(X.abs(), V.abs().t().contiguous()) + U * v.abs()
    ed, ea = eg + 16 * U * (1 + g.abs()), 1.13 * eg + 16 * U * (1 + g * g) * a.abs() + 2 * U * g.abs()
    part = 3 * 2.0 ** -17
    fg = D.abs() * (ev * d.abs() + v.abs() * ed) + (part + 4 * U) * dg.abs()
    fv = D.abs() * ea + (part + 4 * U) * dv.abs()
    w2, w3 = 4 * math.sqrt(2 * N) * U, 4 * math.sqrt(max(1, M)) * U
    e = {"dx": torch.mm(fg + w2 * dg.abs(), G.abs()) + torch.mm(fv + w2 * dv.abs(), V.abs()),
         "dwg": torch.mm((fg + w3 * dg.abs()).t().contiguous(), X.abs()), "dwv": torch.mm((fv + w3 * dv.abs()).t().contiguous(), X.abs())}
    return ref, e


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 64, 40), (40, 384, 96), (300, 333, 301), (777, 512, 130), (5000, 392, 1030)], ids=str)
@pytest.mark.parametrize("act", ["none", "silu"])
def test_gated_gradients_are_rounded_once(device, dtype, shape, act):
    """dx and the weights' gradients of 16-bit data to half a step of it and the products' fp32 roundings: nothing on the way
    is rounded to the data's type."""
    M, K, N = shape
    dt = TYPES[dtype]
    x, dh = randn(device, (M, K), 501, dtype=dt), randn(device, (M, N), 502, dtype=dt)
    wg, wv = (randn(device, (N, K), 503 + i, K ** -0.5, dtype=dt) for i in range(2))
    ref, e = ff_back_bounds(x, wg, wv, act, dh)
    for name, got in zip(("dx", "dwg", "dwv"), stx.gated_ff_back(dh, x, wg, wv, ACTS[act])):
        close(got, ref[name], e[name], name)


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("small", [False, True])
def test_gated_gradients_of_scaled_halves(device, small, aligned):
    """fp16 with the loss scaled: gradients of the two products beyond 65,504 and below 2^-25, sums of them in range."""
    M, K, N = 400, 72 if aligned else 71, 88
    dt = torch.float16
    if small:
        x, dh = randn(device, (M, K), 511, 200.0, dtype=dt), randn(device, (M, N), 512, 2.0 ** -17, dtype=dt)
        wg, wv = (randn(device, (N, K), 513 + i, 2.0 ** -22, dtype=dt) for i in range(2))
    else:
        x, dh = randn(device, (M, K), 515, 2.0 ** -6, dtype=dt), randn(device, (M, N), 516, 6000.0, dtype=dt)
        wg, wv = randn(device, (N, K), 517, 2.0 ** -14, dtype=dt), randn(device, (N, K), 518, 100.0, dtype=dt)
        wv[:, ::2] = 0
    ref, e = ff_back_bounds(x, wg, wv, "none", dh)
    X, G, V, D = (t.to(F64) for t in (x, wg, wv, dh))
    dg = D * torch.mm(X, V.t().contiguous())
    assert bool((dg.abs() < 2.0 ** -25).any() if small else (dg.abs() > 65504).any())
    fits = {n: ref[n].abs() < 65000 for n in e}
    assert float(fits["dwg"].double().mean()) > 0.9 and (small or float(fits["dx"][:, ::2].double().mean()) > 0.9)
    for name, got in zip(("dx", "dwg", "dwv"), stx.gated_ff_back(dh, x, wg, wv, stx.ACT_NONE)):
        keep = fits[name]
        close(got[keep], ref[name][keep], e[name][keep], name)


# ------------------------------------------------------------------- gated block, fp32 products
def bits(device, *values):
    return torch.tensor(values, dtype=torch.int32, device=device).view(torch.float32)


@pytest.mark.parametrize("K", [1, 2, 3, 4])
def test_gated_fp32_products_of_long_mantissas(device, K):
    """Products of fp32 values whose low 16 bits are all ones, all alike in sign, with a value product of 1: the bf16
    parts leave out less than u of each, its sums round it twice. 4 u in all."""
    M, N = 130, 24
    worst = bits(device, 0x3F80FFFF, 0x3F81FFFF, 0x3FFFFFFF, 0x3F80FFFD)
    g = torch.Generator(device=device)
    g.manual_seed(520)
    pick = lambda *s: worst[torch.randint(0, 4, s, generator=g, device=device)]  # noqa: E731
    x, w = pick(M, K), pick(N, K)
    x[0], w[0] = worst[0], worst[0]
    one = torch.ones(N, device=device)
    h = stx.gated_ff(x, w, torch.zeros_like(w), stx.ACT_NONE, b_value=one)
    want = torch.mm(x.to(F64), w.to(F64).t().contiguous())
    assert float(((h.to(F64) - want).abs() / want).max()) <= 4 * U
    # The largest finite values have no part beyond them.
    top = bits(device, 0x7F7FFFFF).expand(M, K).contiguous()
    h = stx.gated_ff(top, torch.full_like(w, 2.0 ** -4), torch.zeros_like(w), stx.ACT_NONE, b_value=one)
    want = (top.to(F64).sum(1) * 2.0 ** -4)[:, None].expand(M, N)
    assert float(((h.to(F64) - want).abs() / want).max()) <= 4 * U


def test_gated_fp32_products_are_unbiased(device):
    """Positive operands: the errors' mean lies within six standard errors of 0, taken over the 512 independent rows of
    the weights (an error that is always towards zero lies at 0.7 u)."""
    M, K, N = 640, 256, 512
    g = torch.Generator(device=device)
    g.manual_seed(521)
    x, w = (torch.rand(s, generator=g, device=device) + 0.5 for s in ((M, K), (N, K)))
    h = stx.gated_ff(x, w, torch.zeros_like(w), stx.ACT_NONE, b_value=torch.ones(N, device=device))
    want = torch.mm(x.to(F64), w.to(F64).t().contiguous())
    e = (h.to(F64) - want) / want
    assert abs(float(e.mean())) <= 6 * float(e.square().mean().sqrt()) / math.sqrt(N)
    dw = stx.gated_ff_back(torch.ones(M, N, device=device), x, w, torch.zeros_like(w), stx.ACT_NONE, b_value=torch.ones(N, device=device))[1]
    want = x.to(F64).sum(0).expand(N, K)                      # one row for all n: 256 independent columns
    e = ((dw.to(F64) - want) / want)[0]
    assert abs(float(e.mean())) <= 6 * float(e.square().mean().sqrt()) / math.sqrt(K)


# ------------------------------------------------------------------------------- streams
def test_outputs_belong_to_the_given_stream(device):
    """With a stream that is not the current one, what a call makes comes from that stream's memory, to which it goes back
    once dropped."""
    s = torch.cuda.Stream()
    x, w = randn(device, (300, 64), 531), randn(device, (96, 64), 532, 0.125)
    pos = torch.arange(300, device=device, dtype=torch.int32)
    want = stx.gated_ff(x, w, w)
    stats = stx.group_norm_cl(x, 4)[1]
    s.wait_stream(torch.cuda.current_stream())

    def owner(t):
        return [g["stream"] for g in torch.cuda.memory_snapshot() if g["address"] <= t.data_ptr() < g["address"] + g["total_size"]]

    assert owner(want) == [torch.cuda.current_stream().cuda_stream]
    for make in (lambda: [stx.gated_ff(x, w, w, stream=s)], lambda: stx.group_norm_cl(x, 4, stream=s), lambda: stx.group_norm_cl_back(x, x, stats, 4, stream=s),
                 lambda: stx.gated_ff_back(want, x, w, w, stream=s)[:3], lambda: [stx.rope_scaled(x.view(1, 300, 1, 64), pos, stx.rope_params(64), stream=s)]):
        for t in make():
            assert owner(t) == [s.cuda_stream]
    s.synchronize()
    y = stx.gated_ff(x, w, w, stream=s)
    s.synchronize()
    assert torch.equal(y, want)


def test_norm_without_statistics(device):
    x = randn(device, (2, 50, 24), 533)
    y, stats = stx.group_norm_cl(x, 3, stats=False)
    assert stats is None and torch.equal(y, stx.group_norm_cl(x, 3)[0])


# ---------------------------------------------------------------------------- group norm
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("place", [0, 5])
def test_group_norm_cl_statistics_of_nonfinite_groups(device, bad, place):
    """1 / sqrt(var + eps) of a group with a NaN or an infinity is NaN, its mean the sum's. The other
    groups' are what they are without it."""
    x = randn(device, (2, 40, 12), 541)
    clean = stx.group_norm_cl(x, 3, act=stx.ACT_SILU)[1]
    x[0, place, 4] = float(bad)
    y, stats = stx.group_norm_cl(x, 3, act=stx.ACT_SILU)
    assert bool(y[0, :, 4:8].isnan().all())
    assert bool(stats[0, 1, 1].isnan()) and torch.equal(stats[0, 1, 0], x[0, :, 4:8].to(F64).mean()) != (bad == "nan")
    stats[0, 1] = clean[0, 1]
    assert torch.equal(stats, clean)


@pytest.mark.parametrize("shape", [(2, 400, 32, 2), (1, 3001, 48, 1), (3, 9, 33, 3), (1, 700, 2048, 512)], ids=str)
@pytest.mark.parametrize("mean,std", [(1e6, 0.25), (-3e5, 0.1), (1e4, 1e-2)])
def test_group_norm_cl_of_small_deviations(device, shape, mean, std):
    """Means of 10^6 and more deviations: the statistics to 1e-10, as of any other data, and the output to the float
    roundings of x - mean. The first token of one slice is 0, which the sums are then taken from."""
    B, T, C, G = shape
    x = randn(device, (B, T, C), 551, std, mean)
    x[0, 0] = 0.0
    w, b = randn(device, (C,), 552, 0.3, 1.0), randn(device, (C,), 553)
    y, stats = stx.group_norm_cl(x, G, 1e-5, w, b)
    ref = norm_ref(x, G, 1e-5, w, b, "none")
    assert torch.allclose(stats, ref["stats"], rtol=1e-10, atol=1e-13)
    close(y, ref["y"], ref["ey"], "y")
    if B > 1:
        ws = torch.empty(stx.group_norm_cl_workspace_size(x, G), dtype=torch.uint8, device=device)
        again, s2 = stx.group_norm_cl(x, G, 1e-5, w, b, out=x, workspace=ws)      # in place: the first elements are overwritten
        assert torch.equal(again, y) and torch.equal(s2, stats)


# ---------------------------------------------------------------------------- activations
# fp32, from the evaluations: 2^y and the reciprocal 1 ulp (2 u) each, the polynomial of GELU 2 u, products and sums u
# each. GELU: q = exp(-z^2/4) within 5 u twice, the rest 6 u: 16 u. Sigmoid: exp(-z) within 5 u, and 4 u: 9 u; SiLU 10 u; 1 - s
# within 16 u on either side. Results below 2^-126 come from subnormal factors, each rounded to 2^-150, times |z| < 16.
TINY = 16 * 2.0 ** -149


def grid(device, act, top=12.0):
    z = torch.linspace(-14.3 if act == "gelu" else -86.0, top, 60000, dtype=F64, device=device).to(torch.float32)
    return torch.cat([z, -torch.logspace(-30, 0, 500, device=device), torch.tensor([0.0, 1e30, -1e30, -200.0, 200.0], device=device)])


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("act,most", [("gelu", 16), ("silu", 10), ("sigmoid", 9)])
def test_fp32_activations_in_the_tails(device, few, act, most):
    """act(z) in fp32 to a few u of itself, wherever it is small: z as one token's gate products, or as many tokens'."""
    z, one = grid(device, act), torch.ones(1, 1, device=device)
    x, w = (one, z[:, None]) if few else (z[:, None], one)
    h = stx.gated_ff(x, w, torch.zeros_like(w), ACTS[act], b_value=torch.ones_like(w[:, 0])).flatten()
    want = act_ref(z.to(F64).clamp_min(-1000), act)[0]
    off = ((h.to(F64) - want).abs() - TINY).clamp_min(0)
    assert bool((off <= most * U * want.abs()).all()), (float((off / want.abs().clamp_min(TINY)).max()) / U, float(z[(off / want.abs().clamp_min(TINY)).argmax()]))


@pytest.mark.parametrize("op", ["norm", "gated"])
@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid"])
def test_fp32_slopes_in_the_tails(device, op, act):
    """act'(z) in fp32, as the bias's gradient of one token: the same bounds of its factors."""
    z = grid(device, act, 40.0)
    n = z.numel()
    if op == "norm":
        stats = torch.tensor([[[0.0, 1.0]]], dtype=F64, device=device)             # xhat is x
        d = stx.group_norm_cl_back(torch.ones(1, n, device=device), z[None], stats, 1, act=ACTS[act])[2]
    else:
        d = stx.gated_ff_back(torch.ones(1, n, device=device), torch.ones(1, 1, device=device), z[:, None], torch.zeros(n, 1, device=device), ACTS[act],
                              torch.zeros(n, device=device), torch.ones(n, device=device))[3]
    y = z.to(F64).clamp(-1000, 1000)
    want = act_ref(y, act)[1]
    s, r = torch.sigmoid(y), torch.sigmoid(-y)
    scale = {"gelu": 16 * (0.5 * torch.erfc(-y / math.sqrt(2.0)) + y.abs() * torch.exp(-y * y / 2) * 0.4), "sigmoid": 26 * s * r, "silu": 26 * s * (1 + y.abs() * r)}[act]
    off = ((d.to(F64) - want).abs() - TINY).clamp_min(0)
    assert bool((off <= U * scale).all()), (float((off / scale.clamp_min(TINY)).max()) / U, float(z[(off / scale.clamp_min(TINY)).argmax()]))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_half_slopes_of_open_gates(device, dtype):
    """The slope of a sigmoid near 1 keeps its digits in 16-bit data too: 26 u and the exponent's |z| u."""
    z = torch.linspace(-30, 30, 2001, device=device).to(TYPES[dtype])
    n, dt = z.numel(), TYPES[dtype]
    d = stx.gated_ff_back(torch.ones(1, n, device=device, dtype=dt), torch.ones(1, 1, device=device, dtype=dt), z[:, None], torch.zeros(n, 1, device=device, dtype=dt),
                          stx.ACT_SIGMOID, torch.zeros(n, device=device), torch.ones(n, device=device))[3]
    want = act_ref(z.to(F64), "sigmoid")[1]
    assert bool(((d.to(F64) - want).abs() <= (26 + z.to(F64).abs()) * U * want).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [1e24, 1e-22])
def test_group_norm_cl_gradient_at_the_ranges_ends(device, dtype, scale):
    """Data whose variance lies beyond fp32 (and without eps below it): the gradients of the same data at scale 1, bound
    and all, divided by the scale."""
    dt = TYPES[dtype]
    x, dy = (randn(device, (2, 60, 24), 561 + i, scale if i == 0 else 1.0, dtype=dt) for i in range(2))
    w, b = randn(device, (24,), 563, 0.3, 1.0), randn(device, (24,), 564, 0.3)
    ref = norm_ref(x, 3, 0.0, w, b, "silu", dy)
    y, stats = stx.group_norm_cl(x, 3, 0.0, w, b, stx.ACT_SILU)
    close(y, ref["y"], ref["ey"], "y")
    dx, dw, db = stx.group_norm_cl_back(dy, x, stats, 3, w, b, stx.ACT_SILU)
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        close(got, ref[name], ref["e" + name], name)


# ------------------------------------------------------------------------------- large calls
def test_group_norm_cl_of_more_slices_than_a_launch_has_blocks(device):
    """2^24 slices and a few of one token: a workgroup each, more than a launch may have."""
    B, C = (1 << 24) + 3, 8
    x = randn(device, (B, 1, C), 571, dtype=torch.bfloat16)
    y, stats = stx.group_norm_cl(x, 2, act=stx.ACT_SILU)
    dx, dw, db = stx.group_norm_cl_back(x, x, stats, 2, act=stx.ACT_SILU)
    sums = torch.zeros(2, C, dtype=F64, device=device)
    bound = torch.zeros(2, C, dtype=F64, device=device)
    for part in torch.arange(B, device=device).split(1 << 21):
        s = slice(int(part[0]), int(part[-1]) + 1)
        v = x[s].view(-1, 2, 4)                                                   # a group is a slice of its own
        ref = norm_ref(v.reshape(-1, 4, 1), 1, 1e-5, None, None, "silu", v.reshape(-1, 4, 1))
        close(y[s].view(-1, 4, 1), ref["y"], ref["ey"], "y")
        close(dx[s].view(-1, 4, 1), ref["dx"], ref["edx"], "dx")
        assert torch.allclose(stats[s].view(-1, 1, 2), ref["stats"], rtol=1e-10, atol=1e-13)
        z = (v.to(F64) - ref["stats"][:, 0, 0].view(-1, 2, 1)) * ref["stats"][:, 0, 1].view(-1, 2, 1)
        d = v.to(F64) * act_ref(z, "silu")[1]
        e = (64 * U * (1 + z.abs()) * v.to(F64).abs()).flatten(1)
        sums += torch.stack([(d * z).flatten(1).sum(0), d.flatten(1).sum(0)])
        bound += torch.stack([(e * (1 + z.abs().flatten(1))).sum(0), e.sum(0)])
    close(dw, sums[0], bound[0], "dw")
    close(db, sums[1], bound[1], "db")


def test_rope_of_more_tokens_than_a_launch_has_blocks(device):
    """2^24 tokens and a few, a workgroup each (rows of odd halves, element by element), in place: the first and the last."""
    N, H, D = (1 << 24) + 3, 2, 514
    q = torch.zeros(1, N, H, D, dtype=torch.bfloat16, device=device)
    at = [0, 1, (1 << 23) - 1, 1 << 23, (1 << 24) - 1, 1 << 24, N - 1]
    x = randn(device, (1, len(at), H, D), 572, dtype=torch.bfloat16)
    q[:, at] = x
    pos = torch.arange(N, device=device, dtype=torch.int32)
    stx.rope_scaled(q, pos, stx.rope_params(D, 2), out=q)
    want, mag = rope_ref(x, pos[at], D, 2)
    close(q[:, at], want, 4 * U * mag, "rope")
    del q
    torch.cuda.empty_cache()


def test_group_norm_cl_in_its_smaller_workspace(device):
    """The forward call in exactly what its own query asks for: the same bits, and nothing beyond written."""
    for shape, G in (((700, 1, 24), 8), ((3, 4001, 48), 1), ((1, 2000, 1024), 512)):
        x = randn(device, shape, 581, dtype=torch.bfloat16)
        need = stx.group_norm_cl_forward_workspace_size(x, G)
        room = torch.full((need + 4096,), 77, dtype=torch.uint8, device=device)
        y, stats = stx.group_norm_cl(x, G, workspace=room[:need])
        assert bool((room[need:] == 77).all())
        full = torch.empty(stx.group_norm_cl_workspace_size(x, G), dtype=torch.uint8, device=device)
        want, s2 = stx.group_norm_cl(x, G, workspace=full)
        assert torch.equal(y, want) and torch.equal(stats, s2)


def test_group_norm_cl_gradient_past_32_bits(device):
    """Slices of 2^31 bytes and more: dx of the second one's first, last and other rows, dweight and dbias against 64 bits. All
    but every thousandth row of x and dy are 0, so the sums are those rows'; rows between them have a gradient too."""
    B, T, C, G, step, dt = 2, 1100000, 1024, 4, 1000, torch.bfloat16
    x, dy = (torch.zeros(B, T, C, dtype=dt, device=device) for _ in range(2))
    for i in range(B):
        x[i, ::step] = randn(device, (T // step, C), 591 + i, 1.0, 0.5, dtype=dt)
        dy[i, ::step] = randn(device, (T // step, C), 593 + i, 1.0, 1.0, dtype=dt)
    w, b = randn(device, (C,), 595, 0.3, 1.0), randn(device, (C,), 596, 0.3)
    stats = stx.group_norm_cl(x, G, 1e-5, w, b, stx.ACT_SILU)[1]
    dx = torch.full_like(x, float("nan"))
    dw, db = stx.group_norm_cl_back(dy, x, stats, G, w, b, stx.ACT_SILU, dx=dx)[1:]
    W, bias, n = w.to(F64).view(G, C // G), b.to(F64).view(G, C // G), T * (C // G)
    sums, bounds = torch.zeros(2, C, dtype=F64, device=device), torch.zeros(2, C, dtype=F64, device=device)
    for i in range(B):
        v, g = (t[i, ::step].to(F64).view(-1, G, C // G) for t in (x, dy))
        mean = v.sum((0, 2), keepdim=True) / n
        r = (v.square().sum((0, 2), keepdim=True) / n - mean * mean + 1e-5).rsqrt()
        assert torch.allclose(stats[i], torch.cat([mean, r]).view(2, G).t(), rtol=1e-10, atol=1e-13)

        def slope(v):
            xh = (v - mean) * r
            z = xh * W + bias
            return xh, act_ref(z, "silu")[1], 8 * U * ((xh * W).abs() + bias.abs()) + 32 * U * (1 + z.abs())

        xh, d, ed = slope(v)
        dz, edz = g * d, g.abs() * ed
        s1, s2 = (W * dz).sum((0, 2), keepdim=True) / n, (W * dz * xh).sum((0, 2), keepdim=True) / n
        e1 = (W.abs() * edz).sum((0, 2), keepdim=True) / n
        e2 = (W.abs() * (edz * xh.abs() + 8 * U * dz.abs() * (xh.abs() + 1))).sum((0, 2), keepdim=True) / n
        for rows in (slice(0, T, step), slice(1, T, 99991), slice(T - 3, T)):
            v, g = (t[i, rows].to(F64).view(-1, G, C // G) for t in (x, dy))
            xr, dr, er = slope(v)
            wdz = W * g * dr
            want = r * (wdz - s1 - xr * s2)
            bound = r * ((W * g).abs() * er + e1 + e2 * xr.abs() + 8 * U * (wdz.abs() + s1.abs() + (xr * s2).abs() + s2.abs()))
            close(dx[i, rows].view(-1, G, C // G), want, bound, f"dx of slice {i}, rows {rows}")
        sums += torch.stack([(dz * xh).sum(0).flatten(), dz.sum(0).flatten()])
        bounds += torch.stack([(edz * xh.abs() + 8 * U * dz.abs() * (xh.abs() + 1)).sum(0).flatten(), (edz + 4 * U * dz.abs()).sum(0).flatten()])
    close(dw, sums[0], bounds[0], "dw")
    close(db, sums[1], bounds[1], "db")
    assert not bool(dx[1].isnan().any())
    del x, dy, dx
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ slices of one buffer
def test_outputs_beside_inputs_in_one_buffer(device):
    """Slices whose rows alternate in memory share no element: taken, with the bits of separate tensors and the rest of the
    buffer as it was."""
    dt = torch.bfloat16
    room = randn(device, (150, 100), 601, dtype=dt)
    x, out = room[:, :40], room[:, 60:84]
    wg, wv = (randn(device, (24, 40), 602 + i, 0.2, dtype=dt) for i in range(2))
    before, want = room.clone(), stx.gated_ff(x.contiguous(), wg, wv)
    stx.gated_ff(x, wg, wv, out=out)
    assert torch.equal(out, want) and torch.equal(room[:, :60], before[:, :60]) and torch.equal(room[:, 84:], before[:, 84:])
    dh = randn(device, (150, 24), 604, dtype=dt)
    grads = stx.gated_ff_back(dh, x, wg, wv)
    both = torch.zeros(24, 80, device=device, dtype=dt)
    got = stx.gated_ff_back(dh, x, wg, wv, dw_gate=both[:, :40], dw_value=both[:, 40:])
    assert all(torch.equal(a, b) for a, b in zip(got[:3], grads[:3]))
    qkv = randn(device, (2, 30, 12, 16), 605, dtype=dt)
    pos = torch.arange(30, device=device, dtype=torch.int32)
    q, k = qkv[:, :, :4], qkv[:, :, 4:6]
    yq, yk = stx.rope_scaled(q, pos, stx.rope_params(16), k)
    copy = qkv.clone()
    stx.rope_scaled(copy[:, :, :4], pos, stx.rope_params(16), copy[:, :, 4:6], out=copy[:, :, 6:10], k_out=copy[:, :, 10:])   # into the rows beside
    assert torch.equal(copy[:, :, 6:10], yq) and torch.equal(copy[:, :, 10:], yk) and torch.equal(copy[:, :, :6], qkv[:, :, :6])
    turned = torch.empty(4, 30, 2, 16, device=device, dtype=dt).permute(2, 1, 0, 3)                                           # heads outermost
    assert torch.equal(stx.rope_scaled(q, pos, stx.rope_params(16), out=turned), yq)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("N", [8, 7])
def test_gated_gradients_of_infinite_and_largest_gradients(device, dtype, N):
    """An infinite dh makes infinite what it enters, by the sign of the weight or token that it meets, and no NaN; the largest
    finite gradients of the products stay finite."""
    M, K, dt = 70, 24, TYPES[dtype]
    x = randn(device, (M, K), 611, dtype=dt).abs() + 0.5
    wg = randn(device, (N, K), 612, 0.5, dtype=dt)
    wg = torch.where(wg.abs() < 0.01, torch.full_like(wg, 0.25), wg)
    dh = randn(device, (M, N), 613, dtype=dt)
    dh[5, 3] = float("inf")
    one = torch.ones(N, device=device)
    dx, dwg, dwv, _, _ = stx.gated_ff_back(dh, x, wg, wg.clone(), stx.ACT_NONE)      # both products are g: dg = dv = dh g
    g = torch.mm(x[5:6].to(F64), wg[3:4].to(F64).t().contiguous()).sign()
    assert torch.equal(dx[5].to(F64), math.inf * g[0] * wg[3].to(F64).sign())
    assert torch.equal(dwg[3].to(F64), math.inf * g.expand(1, K)[0]) and torch.equal(dwv[3], dwg[3])
    keep = torch.arange(M, device=device) != 5
    assert bool(dx[keep].isfinite().all()) and bool(dwg[[0, 1, 2, 4, 5, 6]].isfinite().all())
    if dtype == "bf16":
        dh = torch.zeros_like(dh)
        dh[0, 0] = torch.finfo(dt).max
        w = torch.full_like(wg, 2.0 ** -12)
        dx = stx.gated_ff_back(dh, x, w, torch.zeros_like(w), stx.ACT_NONE, torch.zeros_like(one), one * 1.0039)[0]          # dg rounds to infinity as bf16
        want = float(torch.finfo(dt).max) * float(one[0] * 1.0039) * 2.0 ** -12
        assert bool(((dx[0].to(F64) - want).abs() <= half_step(dt) * 1.01 * want).all())


@pytest.mark.parametrize("M", [40, 70])
@pytest.mark.parametrize("K", [24, 23])
def test_gated_fp32_products_of_infinities(device, M, K):
    """Infinite tokens and weights in fp32: what the sums of products are in floating point (an infinity, or NaN with a zero
    or another sign), at 40 tokens as at 70, and the rows that meet none as they are without."""
    N = 30
    x, wg, wv = (randn(device, s, 621 + i) for i, s in enumerate(((M, K), (N, K), (N, K))))
    wv = wv.abs() + 0.1
    clean = stx.gated_ff(x, wg, wv, stx.ACT_NONE)
    x[3, 2], x[5, 1], x[9, 0], x[9, 4], x[11, 7], x[M - 1, K - 1] = math.inf, -math.inf, math.inf, -math.inf, math.nan, math.inf
    wg[1, 3], wg[2, 5], wg[4, 2], wv[6, 9] = math.inf, -math.inf, 0.0, math.inf
    got = stx.gated_ff(x, wg, wv, stx.ACT_NONE)
    want = (x.to(F64)[:, None] * wg.to(F64)).sum(-1) * (x.to(F64)[:, None] * wv.to(F64)).sum(-1)
    assert torch.equal(got.isnan(), want.isnan()) and 5 * N > int(want.isnan().sum()) > N
    assert torch.equal(got[want.isinf()].to(F64), want[want.isinf()]) and int(want.isinf().sum()) > 2 * M
    rows = [m for m in range(M) if m not in (3, 5, 9, 11, M - 1)]
    cols = [n for n in range(N) if n not in (1, 2, 4, 6)]
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])


def test_gated_fp32_gradients_of_infinite_gradients(device):
    for N in (8, 7):
        test_gated_gradients_of_infinite_and_largest_gradients(device, "f32", N)
