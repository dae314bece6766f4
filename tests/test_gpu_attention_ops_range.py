"""The attention operators (diff_attention*.hip) at values far from 1. Bounds are those of test_gpu_attention_ops.py, with what
each test adds to them."""
import math

import pytest

import stx
from test_gpu_attention_ops import check_diff, diff_back_ref, diff_inputs, seen_ref
from test_gpu_layer_ops import F64, TYPES, close, norm_close, randn

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
