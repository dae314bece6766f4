"""Refusals of the attention operators through the C ABI where an output lies over what the call reads beside its tensors. They
come before any device work, so these run without a GPU (the addresses are never dereferenced)."""
import ctypes

import pytest

import stx
from test_layer_ops_refusals import F32, GB, INVALID, L, desc, ref

N, B, D, POS, FACTORS = 10, 2, 64, 8 * GB, 9 * GB


def params():
    p = stx.rope_params(D)
    p.freq_factors = FACTORS
    return p


# Over the first and the last of the positions of B sequences, 100 apart, and of the factors; behind them nothing is refused.
OVER = [POS - 64, POS + 4 * (100 * (B - 1) + N - 1), FACTORS - 64, FACTORS + 4 * (D // 2 - 1)]


@pytest.mark.parametrize("at", OVER)
@pytest.mark.parametrize("side", ["q", "k"])
def test_qk_outputs_over_positions(at, side):
    q, k = desc([D, 4, N, B], GB), desc([D, 2, N, B], 2 * GB)
    dq, dk = desc([D, 4, N, B], at if side == "q" else 3 * GB), desc([D, 2, N, B], at if side == "k" else 4 * GB)
    assert L.stx_qk_norm_rope(ref(q), ref(k), F32, POS, 100, ctypes.byref(params()), None, None, 0, 1e-6, ref(dq), ref(dk), None) == INVALID
    assert b"pos" in L.stx_last_error() or b"freq_factors" in L.stx_last_error()


@pytest.mark.parametrize("at", OVER)
@pytest.mark.parametrize("what", ["dq", "dk", "dw_q", "dw_k", "ws"])
def test_qk_gradients_over_positions(at, what):
    q, k, dyq, dyk = desc([D, 4, N, B], GB), desc([D, 2, N, B], 2 * GB), desc([D, 4, N, B], 3 * GB), desc([D, 2, N, B], 4 * GB)
    o = dict(dq=5 * GB, dk=6 * GB, dw_q=10 * GB, dw_k=11 * GB, ws=12 * GB)
    o[what] = at // 256 * 256 if what == "ws" else at
    dq, dk = desc([D, 4, N, B], o["dq"]), desc([D, 2, N, B], o["dk"])
    assert L.stx_qk_norm_rope_back(ref(dyq), ref(dyk), ref(q), ref(k), F32, POS, 100, ctypes.byref(params()), None, None, 0, 1e-6, ref(dq), ref(dk), o["dw_q"],
                                   o["dw_k"], o["ws"], 1 << 20, None) == INVALID
    assert b"pos" in L.stx_last_error() or b"freq_factors" in L.stx_last_error()


def test_rel_gradient_of_too_many_heads_without_scores():
    """Heads are checked also where there are no scores, for the table's gradient is made for each."""
    none = desc([0, 8, 1 << 16, 1], GB)
    p = stx.rel_params()
    assert L.stx_soft_max_rel_back(ref(none), ref(none), F32, ctypes.byref(p), 1.0, None, None, None, 8 * GB, None, 0, None) == INVALID
    assert b"heads" in L.stx_last_error()
