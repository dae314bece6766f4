"""The attention operators (qk_norm.hip, soft_max_rel.hip, diff_attention*.hip) at values far from 1, in place in short rows, and with
some of their outputs alone. Bounds are those of test_gpu_attention_ops.py, with what each test adds to them."""
import math

import pytest

import stx
from test_gpu_attention_ops import check_diff, diff_back_ref, diff_inputs, diff_maps, qk_back_ref, seen_ref
from test_gpu_layer_ops import F64, TYPES, U, close, half_step, norm_close, randn

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ------------------------------------------------------------------------ differential attention
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hk", [1, 2])
@pytest.mark.parametrize("lams", [(300.0, -300.0), (0.0, 0.0), (257.0, 0.5), (-16384.0, 1.0)])
def test_diff_large_lambda(device, dtype, Hk, lams):
    """Any weight of the second map. A causal first query gives its key all of both maps, so that P1 - lambda P2, which the
    gradient of v multiplies, is as large as it can be. fp16 holds 2^s of it, with s = 8 or what keeps 2^s |lambda| at 2^14,
    to 2^-25 where it is subnormal."""
    B, M, H, D, V = 1, 70, 2, 64, 128
    q, k, v, _, _, _ = diff_inputs(device, TYPES[dtype], (B, M, M, H, Hk, D, V, True, None))
    v *= 0.25
    lam = torch.tensor(lams, device=device)
    dy = randn(device, (B, M, H, V), 7, 0.02, dtype=q.dtype)
    mask, _ = seen_ref(B, M, M, None, None, True, device)
    kept = stx.diff_attention(q, k, v, lam, causal=True, keep=True)
    check_diff(kept, q, k, v, lam, mask, D ** -0.5, "lambda")
    got = stx.diff_attention_back(dy, q, k, v, lam, *kept, causal=True)
    want = diff_back_ref(dy, q, k, v, lam, *kept, mask, D ** -0.5)
    s = 8 - max(0, math.ceil(math.log2(max(1.0, max(abs(x) for x in lams)))) - 6)
    held = 2.0 ** (-25 - s) * dy.to(F64).abs().unflatten(2, (Hk, H // Hk)).sum((1, 3))[:, None] if dtype == "f16" else 0.0
    for g, (w, bound), name in zip(got, want, ("dq", "dk", "dv", "dlam")):
        close(g, w, bound + (held if name == "dv" else 0.0), "lambda " + name)
        if name != "dlam":
            norm_close(g, w, 2, "lambda " + name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("shape", [(3, 1, 300, 8, 2, 64, 128), (3, 70, 300, 4, 2, 64, 128), (3, 6, 90, 2, 1, 128, 256), (3, 140, 200, 2, 1, 33, 47)],
                         ids=lambda s: "-".join(map(str, s)))
def test_diff_what_causality_hides(device, dtype, what, shape):
    """Keys behind a sequence's last query (a cache that is not filled yet, without lengths) and queries that see no key hold anything."""
    B, M, N, H, Hk, D, V = shape
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (*shape, False, None))
    dy = randn(device, (B, M, H, V), 7, dtype=q.dtype)
    starts = torch.tensor([N // 3, 0, -(M // 2) - 1], device=device, dtype=torch.int32)
    results = []
    for fill in (0.0, what):
        for b, at in enumerate(starts.tolist()):
            k[b, max(0, at + M):] = v[b, max(0, at + M):] = fill
            q[b, :max(0, -at)] = dy[b, :max(0, -at)] = fill
        kept = stx.diff_attention(q, k, v, lam, causal=True, starts=starts, keep=True)
        results.append([*kept, *stx.diff_attention_back(dy, q, k, v, lam, *kept, causal=True, starts=starts)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert bool((results[1][3][2, :M // 2 + 1] == 0).all())


def back_of(part, got, dy, q, k, v, lam, kept, mask, scale, what):
    """dq, dk and dv against those of these operands alone; dk and dv of the keys `part`."""
    want = diff_back_ref(dy, q, k, v, lam, *kept, mask, scale)
    for g, (w, bound), name in zip(got, want, ("dq", "dk", "dv")):
        w, bound = (t[:, part] if name != "dq" else t for t in (w, bound))
        close(g, w, bound, f"{what} {name}")
        norm_close(g, w, 2, f"{what} {name}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lowered", ["dy", "v"])
def test_diff_back_of_a_quiet_sequence(device, dtype, lowered):
    """A sequence whose dy, or v, is 2^16 or 2^13 times smaller than another's of the batch has the accuracy that it has alone."""
    B, M, N, H, Hk, D, V = 2, 200, 200, 2, 1, 64, 128
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (B, M, N, H, Hk, D, V, False, None))
    dy = randn(device, (B, M, H, V), 7, 1.0)
    if lowered == "dy":
        dy[0] *= 2.0 ** 10
        dy[1] *= 2.0 ** -6
    else:
        v[0] *= 2.0 ** 9
        v[1] *= 2.0 ** -4
    dy = dy.to(q.dtype)
    kept = stx.diff_attention(q, k, v, lam, keep=True)
    got = stx.diff_attention_back(dy, q, k, v, lam, *kept)
    mask = torch.ones(1, M, N, dtype=torch.bool, device=device)
    back_of(slice(None), [t[1:] for t in got[:3]], dy[1:], q[1:], k[1:], v[1:], lam, [t[1:] for t in kept], mask, D ** -0.5, "quiet")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_diff_back_of_a_quiet_key_head(device, dtype):
    """A key head whose values are 2^13 times smaller than its neighbour's."""
    B, M, N, H, Hk, D, V = 1, 200, 200, 4, 2, 64, 128
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (B, M, N, H, Hk, D, V, False, None))
    v[:, :, 0] *= 2.0 ** 9
    v[:, :, 1] *= 2.0 ** -4
    dy = randn(device, (B, M, H, V), 7, dtype=q.dtype)
    kept = stx.diff_attention(q, k, v, lam, keep=True)
    got = stx.diff_attention_back(dy, q, k, v, lam, *kept)
    mask = torch.ones(B, M, N, dtype=torch.bool, device=device)
    of = lambda t, heads: t[:, :, heads:]  # noqa: E731
    back_of(slice(None), [of(got[0], 4), of(got[1], 2), of(got[2], 1)], of(dy, 2), of(q, 4), of(k, 2), of(v, 1), lam[2:],
            [of(kept[0], 2), of(kept[1], 2), kept[2][:, 2:]], mask, D ** -0.5, "head")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,quiet", [(200, 90), (700, 290)])
def test_diff_back_of_quiet_last_rows(device, dtype, M, quiet):
    """The last queries of a causal sequence have gradients 2^16 times smaller than the others: the blocks of 64 keys that only
    they see, and their own dq, keep the accuracy that those rows alone give."""
    B, H, Hk, D, V = 1, 2, 1, 64, 128
    first = M - quiet
    keys = (first + 16 + 63) // 64 * 64
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (B, M, M, H, Hk, D, V, True, None))
    dy = randn(device, (B, M, H, V), 7, 2.0 ** 10)
    dy[:, first:] *= 2.0 ** -16
    dy = dy.to(q.dtype)
    kept = stx.diff_attention(q, k, v, lam, causal=True, keep=True)
    got = stx.diff_attention_back(dy, q, k, v, lam, *kept, causal=True)
    mask, _ = seen_ref(B, M, M, None, None, True, device)
    of = lambda t: t[:, first:]  # noqa: E731
    back_of(slice(keys, None), [of(got[0]), got[1][:, keys:], got[2][:, keys:]], of(dy), of(q), k, v, lam, [of(kept[0]), of(kept[1]), kept[2][..., first:]],
            mask[:, first:], D ** -0.5, "rows")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(24, 801, 801, 4, 4), (4096, 1, 70, 4, 1), (24, 400, 300, 4, 1)], ids=lambda s: "-".join(map(str, s)))
def test_diff_lambda_gradient_is_odd(device, dtype, shape):
    """-dy gives -dlambda. Its share of a row is a mean of dP by the second map, of products each rounded by less than an ulp of dP;
    over the rows of a head such roundings are a walk, 2 sqrt(rows) u of the mean share, unless they all go one way, as the matrix
    instructions' do. 4 u |dlambda| are the results'."""
    B, M, N, H, Hk = shape
    D, V = 64, 128
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (*shape, D, V, False, None))
    dy = randn(device, (B, M, H, V), 7, dtype=q.dtype)
    kept = stx.diff_attention(q, k, v, lam, keep=True)
    one, other = (stx.diff_attention_back(y, q, k, v, lam, *kept)[3].to(F64) for y in (dy, -dy))
    few = slice(0, max(1, 500 // M))
    p, _, _, _, _, v64 = diff_maps(q[few], k[few], v[few], torch.ones(q[few].shape[0], M, N, dtype=torch.bool, device=device), D ** -0.5)
    dp = torch.matmul(dy[few].to(F64).transpose(1, 2).contiguous(), v64.transpose(2, 3).contiguous())
    share = (p[1] * dp.abs()).sum(-1).mean((0, 2))
    assert bool(((one + other).abs() <= 2 * math.sqrt(B * M) * U * share + 4 * U * one.abs()).all()), (one + other).tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 40, 150])
def test_diff_large_scores(device, dtype, M):
    """Scaled scores of up to 2^26, of which fp32 keeps so few digits that a row is nearly one key's: the maps stay maps (outputs
    within sqrt(2) times the largest value) and lse follows the largest score."""
    B, N, H, Hk, D, V = 1, 300, 2, 1, 64, 128
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (B, M, N, H, Hk, D, V, False, None))
    q, k = q * 2.0 ** 10, k * 2.0 ** 10
    mask = torch.ones(B, M, N, dtype=torch.bool, device=device)
    scale = 2.0 ** 25.9 / float(diff_maps(q, k, v, mask, 1.0)[2].max())
    out, second, lse = stx.diff_attention(q, k, v, lam, scale=scale, keep=True)
    top = float(v.to(F64).abs().max()) * math.sqrt(2)
    assert float(second.to(F64).abs().max()) <= top and float(out.to(F64).abs().max()) <= top * (1 + float(lam.abs().max()))
    _, want, size, _, _, _ = diff_maps(q, k, v, mask, scale)
    assert bool(((lse.to(F64) - want).abs() <= ((D + 8) * U * size.squeeze(-1).permute(1, 2, 0, 3) + 4 * U * want.abs())).all())


@pytest.mark.parametrize("dtype,size", [("f32", 1e-25), ("f32", 1e-6), ("bf16", 1e-25), ("bf16", 1e-6), ("bf16", 1e20), ("f16", 1e-3), ("f16", 3e3)])
def test_diff_back_sizes(device, dtype, size):
    """Gradients of these sizes as they are, a third of the rows a hundredth of the others. Where fp16's results are subnormal
    they are off by 2^-25 at most, a root mean square of 2^-25 / sqrt(3)."""
    B, M, N, H, Hk, D, V = 1, 80, 150, 2, 1, 64, 128
    q, k, v, lam, _, _ = diff_inputs(device, TYPES[dtype], (B, M, N, H, Hk, D, V, False, None))
    dy = randn(device, (B, M, H, V), 7, size)
    dy[:, ::3] *= 1e-2
    dy, mask = dy.to(q.dtype), torch.ones(B, M, N, dtype=torch.bool, device=device)
    kept = stx.diff_attention(q, k, v, lam, keep=True)
    got = stx.diff_attention_back(dy, q, k, v, lam, *kept)
    want = diff_back_ref(dy, q, k, v, lam, *kept, mask, D ** -0.5)
    for g, (w, bound), name in zip(got, want, ("dq", "dk", "dv", "dlam")):
        close(g, w, bound, "size " + name)
        if name != "dlam" and dtype != "f32":
            low = 2.0 ** -25 * math.sqrt(w.numel() / 3) * 1.2 if dtype == "f16" else 0.0
            assert float((g.to(F64) - w).norm()) <= half_step(g.dtype) * math.sqrt(2 / 3) * 1.2 * float(w.norm()) + low, name


def tensor(t):
    """The C ABI's description of a tensor (batch, tokens, heads, elements), or NULL."""
    import ctypes
    if t is None:
        return None
    d = stx.Tensor()
    d.data = t.data_ptr()
    for i in range(4):
        d.ne[i], d.nb[i] = t.shape[3 - i], t.stride(3 - i) * t.element_size()
    return ctypes.byref(d)


def pointer(t):
    return None if t is None else t.data_ptr()


TYPE = {torch.float32: stx.TYPE_F32, torch.float16: stx.TYPE_F16, torch.bfloat16: stx.TYPE_BF16}


def ask_alone(outputs, want, call, groups):
    """call(outputs, those not asked for None) for each group alone: the bits of the full call, the rest untouched."""
    for group in groups:
        for i, t in enumerate(outputs):
            t.fill_(7.0)
        call([t if i in group else None for i, t in enumerate(outputs)])
        for i, t in enumerate(outputs):
            assert torch.equal(t, want[i]) if i in group else bool((t == 7.0).all()), (group, i)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 90, 700, 4, 2), (1, 700, 90, 2, 1), (40, 130, 150, 4, 4)], ids=["split keys", "split rows", "whole"])
def test_diff_back_outputs_alone(device, dtype, shape):
    B, M, N, H, Hk = shape
    D, V, dt = 64, 128, TYPES[dtype]
    q, k, v, lam, _, _ = diff_inputs(device, dt, (*shape, D, V, True, None))
    dy = randn(device, (B, M, H, V), 7, dtype=dt)
    kept = stx.diff_attention(q, k, v, lam, causal=True, keep=True)
    want = stx.diff_attention_back(dy, q, k, v, lam, *kept, causal=True)
    L, t = stx.lib(), TYPE[dt]
    a = [tensor(x) for x in (dy, q, k, v)]
    ws = torch.empty(L.stx_diff_attention_back_workspace_size(*a[1:], t), dtype=torch.uint8, device=device)
    s = torch.cuda.current_stream().cuda_stream

    def call(o):
        stx.check(L.stx_diff_attention_back(*a, t, lam.data_ptr(), D ** -0.5, 1, None, None, tensor(kept[0]), tensor(kept[1]), kept[2].data_ptr(),
                                            tensor(o[0]), tensor(o[1]), tensor(o[2]), pointer(o[3]), ws.data_ptr(), ws.numel(), s))

    ask_alone([torch.empty_like(x) for x in want], want, call, ({0}, {1, 2}, {3}, {0, 3}, {1, 2, 3}, {0, 1, 2}, set()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("per_head", [False, True])
def test_qk_back_outputs_alone(device, dtype, per_head):
    import ctypes
    B, N, H, Hk, D, dt = 2, 300, 4, 2, 64, TYPES[dtype]
    q, k = randn(device, (B, N, H, D), 1, dtype=dt), randn(device, (B, N, Hk, D), 2, dtype=dt)
    dyq, dyk = randn(device, q.shape, 3, dtype=dt), randn(device, k.shape, 4, dtype=dt)
    wq, wk = (randn(device, (n, D) if per_head else (D,), 5 + n, 0.3, 1.0) for n in (H, Hk))
    pos, p = torch.arange(N, device=device, dtype=torch.int32), stx.rope_params(D)
    full = stx.qk_norm_rope_back(dyq, q, pos, p, wq, dyk, k, wk)
    want = [full[i] for i in (0, 2, 1, 3)]                        # dq, dk, dw_q, dw_k
    L, t = stx.lib(), TYPE[dt]
    a = [tensor(x) for x in (dyq, dyk, q, k)]
    ws = torch.empty(L.stx_qk_norm_rope_back_workspace_size(a[2], a[3], t, D, per_head), dtype=torch.uint8, device=device)
    s = torch.cuda.current_stream().cuda_stream

    def call(o):
        sums = o[2] is not None or o[3] is not None
        stx.check(L.stx_qk_norm_rope_back(*a, t, pos.data_ptr(), 0, ctypes.byref(p), wq.data_ptr(), wk.data_ptr(), per_head, 1e-6, tensor(o[0]), tensor(o[1]),
                                          pointer(o[2]), pointer(o[3]), ws.data_ptr() if sums else None, ws.numel() if sums else 0, s))

    ask_alone([torch.empty_like(x) for x in want], want, call, ({0}, {1}, {2}, {3}, {0, 1}, {2, 3}, {0, 3}, set()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [5, 150, 2500])
def test_rel_back_outputs_alone(device, dtype, N):
    import ctypes
    B, H, M, dt = 3, 2, 70, TYPES[dtype]
    p = stx.rel_params(16, 40)
    y = stx.soft_max_rel(randn(device, (B, H, M, N), 1, dtype=dt), randn(device, (16, H), 2), p)
    dy = randn(device, y.shape, 3, dtype=dt)
    want = stx.soft_max_rel_back(dy, y, p, 0.5)
    L, t = stx.lib(), TYPE[dt]
    ws = torch.empty(L.stx_soft_max_rel_back_workspace_size(tensor(y), t, 16), dtype=torch.uint8, device=device)
    s = torch.cuda.current_stream().cuda_stream

    def call(o):
        stx.check(L.stx_soft_max_rel_back(tensor(dy), tensor(y), t, ctypes.byref(p), 0.5, None, None, tensor(o[0]), pointer(o[1]),
                                          pointer(ws) if o[1] is not None else None, ws.numel() if o[1] is not None else 0, s))

    ask_alone([torch.empty_like(x) for x in want], want, call, ({0}, {1}, set()))


# ------------------------------------------------------------------------- norms and rotation
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 1024, 33])
@pytest.mark.parametrize("x_size,dy_size,eps", [(1e14, 1e25, 1e-6), (1e16, 1e30, 0.0), (1e-10, 1e-30, 0.0), (1e-18, 1e-25, 0.0), (1e25, 1e12, 0.0),
                                                (1e-25, 1e-8, 0.0)])
def test_qk_back_products_that_leave_fp32(device, dtype, D, x_size, dy_size, eps):
    """Rows whose products w dy x are not floats, or below their normal range, while the squares and the gradient are."""
    B, N, H = 2, 9, 3
    x, dy = randn(device, (B, N, H, D), 1, x_size, dtype=TYPES[dtype]), randn(device, (B, N, H, D), 2, dy_size, dtype=TYPES[dtype])
    w, pos = randn(device, (D,), 3, 0.3, 1.0), torch.arange(3, 3 + N, device=device, dtype=torch.int32)
    dx, dw, _, _ = stx.qk_norm_rope_back(dy, x, pos, stx.rope_params(32), w, eps=eps)
    want, bound, dww, dwm = qk_back_ref(dy, x, w, pos, eps, 32, 0)
    close(dx, want, bound, "dx")
    close(dw, dww.sum((0, 1, 2)), (8 + 4 * math.sqrt(B * N * H)) * U * dwm.sum((0, 1, 2)), "dw")


# ------------------------------------------------------------------ softmax with a position bias
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("M", [5, 61, 300])
def test_rel_short_rows_in_place(device, dtype, N, M):
    """Rows shorter than a vector, a lane each: in place the bits of a call into other memory."""
    B, H, dt = 40, 8, TYPES[dtype]
    x, table, p = randn(device, (B, H, M, N), 1, 4.0, dtype=dt), randn(device, (32, H), 2), stx.rel_params()
    want = stx.soft_max_rel(x, table, p)
    for _ in range(3):
        y = x.clone()
        stx.soft_max_rel(y, table, p, out=y)
        assert torch.equal(y, want)
