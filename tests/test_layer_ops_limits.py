"""Workspace sizes and refusals of the transformer-layer operators through the C ABI beyond those of
test_layer_ops_refusals; none reaches a device."""
import pytest

import stx
from test_layer_ops_refusals import BF16, F32, GB, INVALID, L, desc, norm, ref, rope


@pytest.mark.parametrize("ne", [[256, 1, 1, 1 << 20], [257, 1, 1, 1 << 18], [48, 4000, 1, 3], [512, 1344]])
def test_norm_forward_needs_no_room_for_the_gradients(ne):
    """The forward call's workspace holds pairs of sums and a number a group, not one a position of every slice."""
    a = desc(ne, type=BF16)
    fwd, both = L.stx_group_norm_cl_forward_workspace_size(ref(a), BF16, 2), L.stx_group_norm_cl_workspace_size(ref(a), BF16, 2)
    slices = ne[3] if len(ne) > 3 else 1
    assert 0 < fwd < both
    assert norm(a=a, type=BF16, groups=2, nbytes=fwd - 1) == INVALID and b"workspace" in L.stx_last_error()
    if slices > 1000:                    # a pair of doubles for each group in each column tile (17 at most up to 512 columns), and a double a group
        assert fwd <= slices * 2 * (17 * 16 + 8) + 512 and both >= slices * ne[0] * 16 and fwd <= both // 8


def test_norm_forward_workspace_of_bad_arguments():
    assert L.stx_group_norm_cl_forward_workspace_size(None, F32, 2) == 0
    assert L.stx_group_norm_cl_forward_workspace_size(ref(desc([32, 10])), F32, 0) == 0


# -------------------------------------------------------------------------- memory written twice
QKV = {1: 256, 2: 12 * 256, 3: 10 * 12 * 256}           # a projection's rows: 12 heads of 64 floats a token, 10 tokens, 2 sequences


@pytest.mark.parametrize("kw,word", [
    (dict(q_dst=desc([64, 4, 10, 2], 2 * GB, nb={1: 128})), b"rows of the output"),                       # rows half over each other
    (dict(q_dst=desc([64, 4, 10, 2], 2 * GB, nb={2: 512})), b"rows of the output"),
    (dict(q=desc([64, 4, 10, 2], GB, nb=QKV), q_dst=desc([64, 4, 10, 2], GB + 256, nb=QKV)), b"in part"),   # a head further
    (dict(q=desc([64, 4, 10, 2], GB, nb=QKV), q_dst=desc([64, 4, 10, 2], GB + 11 * 256, nb=QKV)), b"in part"),   # into the next token
    (dict(q=desc([64, 4, 10, 2], GB, nb=QKV), k=desc([64, 4, 10, 2], GB + 1024, nb=QKV), q_dst=desc([64, 4, 10, 2], GB + 1024, nb=QKV)), b"other side"),
    (dict(q=desc([64, 4, 10, 2], GB, nb=QKV), k=desc([64, 2, 10, 2], GB + 1024, nb=QKV), q_dst=desc([64, 4, 10, 2], GB, nb=QKV),
          k_dst=desc([64, 2, 10, 2], GB + 512, nb=QKV)), b"other side"),
    (dict(k=desc([64, 4, 10, 2], 4 * GB), k_dst=desc([64, 4, 10, 2], 2 * GB)), b"other side"),               # both to one place
])
@pytest.mark.parametrize("back", [False, True])
def test_rope_outputs_over_other_memory(kw, word, back):
    assert rope(back=back, **kw) == INVALID and word in L.stx_last_error(), L.stx_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(dweight=GB * 6), b"weight"), (dict(dbias=GB * 7), b"bias"), (dict(dweight=GB * 9, dbias=GB * 9 + 64), b"dbias"), (dict(dweight=GB), b"dweight overlaps a"),
    (dict(dbias=2 * GB + 64), b"dbias overlaps dy"), (dict(dx=desc([32, 10, 1, 2], 5 * GB)), b"dx overlaps stats"), (dict(ws=GB), b"workspace overlaps a"),
    (dict(dweight=16 * GB + 256), b"overlaps the workspace"),
])
def test_norm_gradients_over_other_memory(change, word):
    p = dict(dx=desc([32, 10, 1, 2], 4 * GB), dweight=GB * 8, dbias=GB * 9, ws=GB * 16)
    p.update(change)
    rc = L.stx_group_norm_cl_back(ref(desc([32, 10, 1, 2], 2 * GB)), ref(desc([32, 10, 1, 2])), F32, GB * 5, 4, GB * 6, GB * 7, 0, ref(p["dx"]), p["dweight"],
                                  p["dbias"], p["ws"], 1 << 40, None)
    assert rc == INVALID and word in L.stx_last_error(), L.stx_last_error()


@pytest.mark.parametrize("kw,word", [(dict(stats=GB + 64), b"stats overlaps a"), (dict(stats=2 * GB), b"dst overlaps stats"), (dict(ws=2 * GB), b"workspace"),
                                     (dict(ws=GB), b"workspace overlaps a")])
def test_norm_outputs_over_other_memory(kw, word):
    assert norm(**kw) == INVALID and word in L.stx_last_error(), L.stx_last_error()


SIDE = {1: 4 * 48}                                       # rows of 48 floats: two matrices of 24 side by side


@pytest.mark.parametrize("change,word", [
    (dict(db_gate=11 * GB, db_value=11 * GB + 16), b"db_value"), (dict(db_gate=9 * GB), b"b_gate"), (dict(db_value=5 * GB), b"dh"), (dict(ws=GB), b"workspace overlaps x"),
    (dict(dx=desc([24, 10], 7 * GB)), b"dx overlaps dw_gate"), (dict(dwg=desc([24, 8], 7 * GB, nb=SIDE), dwv=desc([24, 8], 7 * GB + 80, nb=SIDE)), b"dw_value"),
    (dict(dwg=desc([24, 8], 7 * GB, nb=SIDE), dwv=desc([24, 8], 7 * GB + 96, nb={1: 4 * 40})), b"dw_value"),      # rows that cannot be told apart
])
def test_ff_gradients_over_other_memory(change, word):
    p = dict(dx=desc([24, 10], 6 * GB), dwg=desc([24, 8], 7 * GB), dwv=desc([24, 8], 8 * GB), db_gate=11 * GB, db_value=12 * GB, ws=10 * GB)
    p.update(change)
    rc = L.stx_gated_ff_back(ref(desc([8, 10], 5 * GB)), ref(desc([24, 10], GB)), ref(desc([24, 8], 2 * GB)), ref(desc([24, 8], 3 * GB)), F32, 9 * GB, 9 * GB + 4096, 2,
                             ref(p["dx"]), ref(p["dwg"]), ref(p["dwv"]), p["db_gate"], p["db_value"], p["ws"], 1 << 20, None)
    assert rc == INVALID and word in L.stx_last_error(), L.stx_last_error()


def test_ff_output_over_a_bias():
    rc = L.stx_gated_ff(ref(desc([24, 10], GB)), ref(desc([24, 8], 2 * GB)), ref(desc([24, 8], 3 * GB)), F32, 4 * GB + 64, None, 2, ref(desc([8, 10], 4 * GB)), None)
    assert rc == INVALID and b"b_gate" in L.stx_last_error()


@pytest.mark.parametrize("kw", [dict(freq_base=float("inf")), dict(freq_scale=float("inf")), dict(attn_factor=float("nan")), dict(ext_factor=float("nan")),
                                dict(ext_factor=1.0, n_ctx_orig=10, beta_fast=float("inf")), dict(ext_factor=1.0, n_ctx_orig=10, beta_slow=float("inf"))])
def test_rope_parameters_that_are_not_finite(kw):
    assert rope(**kw) == INVALID and b"finite" in L.stx_last_error()
