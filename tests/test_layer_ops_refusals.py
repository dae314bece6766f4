"""Refusals of the transformer-layer operators through the C ABI: each call fails its argument checks
before any device work, so these run without a GPU (the addresses are never dereferenced)."""
import ctypes

import pytest

import stx

L = stx.lib()
INVALID, UNSUPPORTED = stx.STATUS_INVALID_ARGUMENT, stx.STATUS_UNSUPPORTED
F32, F16, BF16 = stx.TYPE_F32, stx.TYPE_F16, stx.TYPE_BF16
SIZE = {F32: 4, F16: 2, BF16: 2}
GB = 1 << 30


def desc(ne, addr=GB, type=F32, nb=None):
    d = stx.Tensor()
    d.data = addr
    step = SIZE.get(type, 4)
    for i in range(4):
        d.ne[i] = ne[i] if i < len(ne) else 1
        d.nb[i] = step
        step *= d.ne[i]
    for i, v in (nb or {}).items():
        d.nb[i] = v
    return d


def ref(d):
    return None if d is None else ctypes.byref(d)


def rope(q=None, k=None, type=F32, pos=GB * 8, stride=0, q_dst="same", k_dst="same", back=False, **kw):
    q = desc([64, 4, 10, 2], type=type) if q is None else q
    p = stx.rope_params(kw.pop("n_dims", 64), kw.pop("mode", 0), **{k_: v for k_, v in kw.items() if k_ != "size"})
    if "size" in kw:
        p.size = kw["size"]
    copy = lambda d, at: None if d is None else desc(list(d.ne), at, type)  # noqa: E731
    q_dst = copy(q, 2 * GB) if q_dst == "same" else q_dst
    k_dst = copy(k, 3 * GB) if k_dst == "same" else k_dst
    fn = L.stx_rope_scaled_back if back else L.stx_rope_scaled
    return fn(ref(q), ref(k), type, pos, stride, ctypes.byref(p), ref(q_dst), ref(k_dst), None)


@pytest.mark.parametrize("kw,status", [
    (dict(type=7), INVALID), (dict(n_dims=63), INVALID), (dict(n_dims=66), INVALID), (dict(n_dims=0), INVALID),
    (dict(mode=1), UNSUPPORTED), (dict(mode=8), UNSUPPORTED), (dict(freq_base=0.0), INVALID), (dict(freq_base=float("nan")), INVALID),
    (dict(freq_scale=0.0), INVALID), (dict(freq_scale=-1.0), INVALID), (dict(ext_factor=1.0), INVALID),
    (dict(ext_factor=1.0, n_ctx_orig=10, beta_fast=0.0), INVALID), (dict(ext_factor=1.0, n_ctx_orig=10, freq_base=1.0), INVALID),
    (dict(stride=-1), INVALID), (dict(pos=None), INVALID), (dict(size=8), INVALID),
    (dict(q=desc([64, 4, 10, 2], nb={0: 8})), INVALID), (dict(q=desc([64, 4, 10, 2], nb={1: 6})), INVALID),
    (dict(q=desc([64, 4, 10, 2], nb={2: -4})), INVALID), (dict(q=desc([64, 4, -1, 2])), INVALID),
    (dict(q=desc([64, 4, 10, 2], addr=None)), INVALID), (dict(q=desc([64, 4, 10, 2], addr=GB + 2)), INVALID),
    (dict(q_dst=desc([64, 4, 10, 1])), INVALID), (dict(q_dst=None), INVALID), (dict(q_dst=desc([64, 4, 10, 2], 2 * GB, nb={1: 0})), INVALID),
    (dict(q_dst=desc([64, 4, 10, 2], GB, nb={1: 1024})), INVALID),          # in place, other strides
    (dict(k=desc([64, 2, 10, 2]), k_dst=None), INVALID), (dict(k_dst=desc([64, 2, 10, 2])), INVALID),
    (dict(k=desc([32, 2, 10, 2], 4 * GB)), INVALID), (dict(k=desc([64, 2, 9, 2], 4 * GB)), INVALID), (dict(k=desc([64, 2, 10, 1], 4 * GB)), INVALID),
    (dict(q=desc([64, 1, 1 << 20, 1 << 12])), INVALID),                          # 2^32 tokens
    (dict(q=desc([9000, 1, 1, 1]), n_dims=8194), UNSUPPORTED),
    (dict(q=desc([64, 1 << 25, 1, 1])), INVALID),
])
@pytest.mark.parametrize("back", [False, True])
def test_rope_refusals(kw, status, back):
    assert rope(back=back, **kw) == status, L.stx_last_error()
    assert L.stx_last_error()


def test_rope_null():
    assert L.stx_rope_scaled(None, None, F32, None, 0, None, None, None, None) == INVALID


def norm(a=None, type=F32, groups=4, eps=1e-5, act=0, dst="same", stats=None, ws=GB * 16, nbytes=None):
    a = desc([32, 10, 1, 2], type=type) if a is None else a
    dst = desc(list(a.ne), 2 * GB, type) if dst == "same" else dst
    nbytes = 1 << 40 if nbytes is None else nbytes
    return L.stx_group_norm_cl(ref(a), type, groups, eps, None, None, act, ref(dst), stats, ws, nbytes, None)


@pytest.mark.parametrize("kw", [
    dict(type=2), dict(groups=0), dict(groups=-1), dict(groups=33), dict(a=desc([10, 5]), groups=7),       # groups of 2: the sixth is empty
    dict(eps=-1.0), dict(eps=float("nan")), dict(act=4), dict(act=-1), dict(dst=None), dict(dst=desc([32, 10, 1, 1], 2 * GB)),
    dict(a=desc([32, 10, 1, 2], nb={1: 256})), dict(dst=desc([32, 10, 1, 2], 2 * GB, nb={1: 256})), dict(dst=desc([32, 10, 1, 2], GB + 128)),
    dict(ws=None), dict(nbytes=16), dict(ws=GB * 16 + 128), dict(a=desc([0, 10])), dict(a=desc([32, 10, 1, 2], None)),
    dict(a=desc([32, 1 << 20, 1 << 20, 1])), dict(a=desc([1 << 24, 1, 1, 1]), groups=1),
])
def test_norm_refusals(kw):
    assert norm(**kw) == INVALID, L.stx_last_error()
    assert L.stx_last_error()


def test_norm_many_groups_unsupported():
    assert norm(a=desc([8192, 4]), groups=8192) == UNSUPPORTED


@pytest.mark.parametrize("change", [dict(dy=desc([32, 9, 1, 2], 2 * GB)), dict(dy=desc([32, 10, 1, 2], 2 * GB, nb={2: 4})), dict(dy=None), dict(stats=None),
                                    dict(dx=desc([32, 10, 1, 2], 2 * GB + 64)), dict(dx=desc([32, 10, 1, 2], GB + 64)), dict(ws=None), dict(act=9),
                                    dict(dx=desc([32, 10, 1, 2], 4 * GB, F16))])
def test_norm_back_refusals(change):
    p = dict(dy=desc([32, 10, 1, 2], 2 * GB), a=desc([32, 10, 1, 2]), stats=GB * 5, dx=desc([32, 10, 1, 2], 4 * GB), ws=GB * 16, act=0)
    if "dy" in change and change["dy"] is not None and change["dy"].nb[2] == 4:
        change["dy"].ne[2], change["dy"].ne[1] = 10, 1                          # the same elements, spaced as nothing is
    p.update(change)
    rc = L.stx_group_norm_cl_back(ref(p["dy"]), ref(p["a"]), F32, p["stats"], 4, None, None, p["act"], ref(p["dx"]), None, None, p["ws"], 1 << 40, None)
    assert rc == INVALID and L.stx_last_error()


def test_norm_workspace_size():
    assert L.stx_group_norm_cl_workspace_size(ref(desc([32, 10, 1, 2], None)), F32, 4) > 0
    assert L.stx_group_norm_cl_workspace_size(None, F32, 4) == 0
    assert L.stx_group_norm_cl_workspace_size(ref(desc([32, 10, 1, 2])), F32, 0) == 0


FF = dict(x=desc([24, 10], GB), wg=desc([24, 8], 2 * GB), wv=desc([24, 8], 3 * GB), dst=desc([8, 10], 4 * GB), type=F32, act=2)
FF_BAD = [
    dict(type=9), dict(act=5), dict(x=None), dict(wg=None), dict(wv=None), dict(x=desc([25, 10], GB)), dict(wg=desc([24, 9], 2 * GB)),
    dict(wg=desc([23, 8], 2 * GB)), dict(wv=desc([24, 8, 2], 3 * GB)), dict(x=desc([0, 10], GB)), dict(wg=desc([24, 0], 2 * GB), wv=desc([24, 0], 3 * GB)),
    dict(x=desc([24, 10], GB, nb={0: 2})), dict(x=desc([24, 5, 2], GB, nb={2: 1000})), dict(x=desc([24, 1 << 20, 1 << 11], GB)),
    dict(wg=desc([24, (1 << 20) + 1], 2 * GB), wv=desc([24, (1 << 20) + 1], 3 * GB)), dict(x=desc([24, 10], GB + 2)),
]


@pytest.mark.parametrize("change", FF_BAD + [dict(dst=None), dict(dst=desc([8, 9], 4 * GB)), dict(dst=desc([7, 10], 4 * GB)), dict(dst=desc([8, 10], GB + 40)),
                                             dict(dst=desc([8, 10], 2 * GB + 4)), dict(dst=desc([8, 10], 4 * GB, nb={1: 28}))])
def test_ff_refusals(change):
    p = {**FF, **change}
    rc = L.stx_gated_ff(ref(p["x"]), ref(p["wg"]), ref(p["wv"]), p["type"], None, None, p["act"], ref(p["dst"]), None)
    assert rc == INVALID and L.stx_last_error()


@pytest.mark.parametrize("change", FF_BAD + [
    dict(dh=None), dict(dh=desc([8, 9], 5 * GB)), dict(dx=desc([24, 9], 6 * GB)), dict(dx=desc([24, 10], 6 * GB, nb={1: 0})), dict(dwg=None), dict(dwv=None),
    dict(dwg=desc([24, 7], 7 * GB)), dict(dwv=desc([24, 8], 7 * GB + 32)), dict(dx=desc([24, 10], 5 * GB)), dict(dx=desc([24, 10], GB)),
    dict(dwg=desc([24, 8], 3 * GB)), dict(ws=None), dict(ws=10 * GB + 16), dict(nbytes=100)])
def test_ff_back_refusals(change):
    p = {**FF, "dh": desc([8, 10], 5 * GB), "dx": desc([24, 10], 6 * GB), "dwg": desc([24, 8], 7 * GB), "dwv": desc([24, 8], 8 * GB), "ws": 10 * GB,
         "nbytes": 1 << 40, **change}
    rc = L.stx_gated_ff_back(ref(p["dh"]), ref(p["x"]), ref(p["wg"]), ref(p["wv"]), p["type"], None, None, p["act"], ref(p["dx"]), ref(p["dwg"]),
                             ref(p["dwv"]), None, None, p["ws"], p["nbytes"], None)
    assert rc == INVALID and L.stx_last_error()


def test_ff_workspace_size():
    size = L.stx_gated_ff_back_workspace_size
    assert size(10, 24, 8, F32) > 0 and size(0, 24, 8, BF16) >= 0
    for bad in ((-1, 24, 8, F32), (10, 0, 8, F32), (10, 24, 0, F32), (10, 24, 8, 5), (1 << 31, 24, 8, F32), (10, 1 << 21, 8, F32)):
        assert size(*bad) == 0


def test_parameter_helpers():
    with pytest.raises(TypeError):
        stx.rope_params(64, freq_factors=[1.0])
    p = stx.rope_params(64, 2, n_ctx_orig=4096, ext_factor=1.0)
    assert p.size == ctypes.sizeof(stx.RopeParams) == 48 and (p.mode, p.n_ctx_orig) == (2, 4096)


def test_workspace_of_another_device():
    """A workspace in host memory never reaches a kernel."""
    import torch
    with pytest.raises(ValueError):
        stx._scratch(256, torch.empty(256, dtype=torch.uint8), torch.empty(1, device="meta"), None)


def test_frequency_factors_of_another_device():
    import torch
    q, pos = torch.empty(2, 4, 8), torch.zeros(2, dtype=torch.int32)
    p = stx.rope_params(8)
    p.factors = torch.ones(4, device="meta")
    with pytest.raises(ValueError, match="freq_factors"):
        stx.rope_scaled(q, pos, p)
