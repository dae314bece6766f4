"""The attention operators' Python binding and refusals without a GPU: on which stream it allocates, what it and the C ABI
refuse before any device work (addresses are never dereferenced)."""
import ctypes

import pytest

import stx
from test_layer_ops_binding import Stream, allocations  # noqa: F401  (a fixture)
from test_layer_ops_refusals import BF16, F16, F32, GB, INVALID, L, SIZE, UNSUPPORTED, desc, ref

torch = pytest.importorskip("torch")


def calls(stream):
    q, pos, w = torch.ones(2, 3, 4, 8), torch.arange(3, dtype=torch.int32), torch.ones(8)
    x, table = torch.ones(2, 4, 3, 5), torch.ones(32, 4)
    k, v, lam = torch.ones(2, 5, 4, 8), torch.ones(2, 5, 2, 8), torch.ones(2)
    out, lse = torch.ones(2, 3, 2, 8), torch.ones(2, 2, 2, 3)
    return [
        lambda: stx.qk_norm_rope(q, pos, stx.rope_params(8), w, q, w, stream=stream),
        lambda: stx.qk_norm_rope_back(q, q, pos, stx.rope_params(8), w, q, q, w, stream=stream),
        lambda: stx.soft_max_rel(x, table, stx.rel_params(), stream=stream),
        lambda: stx.soft_max_rel_back(x, x, stx.rel_params(), stream=stream),
        lambda: stx.diff_attention(q, k, v, lam, keep=True, stream=stream),
        lambda: stx.diff_attention_back(out, q, k, v, lam, out, out, lse, stream=stream),
    ]


@pytest.mark.parametrize("call", range(6))
def test_new_tensors_belong_to_the_calls_stream(allocations, call):  # noqa: F811
    stream = Stream()
    for s in (stream, None):
        run = calls(s)[call]
        allocations.clear()
        run()
        assert allocations and all(on is s for _, on in allocations), allocations


def test_nothing_kept_without_keep(allocations):  # noqa: F811
    q, k, v = torch.ones(2, 3, 4, 8), torch.ones(2, 5, 4, 8), torch.ones(2, 5, 2, 8)
    out, second, lse = stx.diff_attention(q, k, v, torch.ones(2))
    assert out.shape == (2, 3, 2, 8) and second is None and lse is None
    _, dtable = stx.soft_max_rel_back(torch.ones(2, 4, 3, 5), torch.ones(2, 4, 3, 5), stx.rel_params(), dtable=False)
    assert dtable is None


def test_binding_refuses():
    q, pos, p = torch.ones(2, 3, 4, 8), torch.arange(3, dtype=torch.int32), stx.rope_params(8)
    with pytest.raises(ValueError, match="w_q"):
        stx.qk_norm_rope(q, pos, p, torch.ones(4))
    with pytest.raises(ValueError, match="w_k"):
        stx.qk_norm_rope(q, pos, p, None, None, torch.ones(8))
    with pytest.raises(ValueError, match="both"):
        stx.qk_norm_rope(q, pos, p, torch.ones(8), q, torch.ones(4, 8))
    with pytest.raises(ValueError, match="pos"):
        stx.qk_norm_rope(q, pos[:2], p)
    with pytest.raises(ValueError, match="table"):
        stx.soft_max_rel(torch.ones(2, 4, 3, 5), torch.ones(16, 4), stx.rel_params())
    with pytest.raises(ValueError, match="queries"):
        stx.soft_max_rel(torch.ones(4, 3, 5), torch.ones(32, 4), stx.rel_params())
    with pytest.raises(ValueError, match="heads"):
        stx.diff_attention(torch.ones(2, 3, 3, 8), torch.ones(2, 5, 4, 8), torch.ones(2, 5, 2, 8), torch.ones(1))
    p = stx.rel_params(64, 1000, False, True)
    assert p.size == ctypes.sizeof(stx.RelParams) == 20 and (p.n_buckets, p.max_distance, p.bidirectional, p.causal) == (64, 1000, 0, 1)


# ------------------------------------------------------------------------- norms and rotation
def qk(q=None, k=None, type=F32, pos=GB * 8, stride=0, q_dst="same", k_dst="same", w_q=GB * 9, w_k=None, per_head=0, eps=1e-6, n_dims=64, mode=0, **kw):
    q = desc([64, 4, 10, 2], type=type) if q is None else q
    p = stx.rope_params(n_dims, mode, **kw)
    copy = lambda d, at: None if d is None else desc(list(d.ne), at, type)  # noqa: E731
    q_dst = copy(q, 2 * GB) if q_dst == "same" else q_dst
    k_dst = copy(k, 3 * GB) if k_dst == "same" else k_dst
    return L.stx_qk_norm_rope(ref(q), ref(k), type, pos, stride, ctypes.byref(p), w_q, w_k, per_head, eps, ref(q_dst), ref(k_dst), None)


@pytest.mark.parametrize("kw,status", [
    (dict(type=7), INVALID), (dict(n_dims=63), INVALID), (dict(n_dims=66), INVALID), (dict(mode=1), UNSUPPORTED), (dict(freq_base=0.0), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(eps=float("inf")), INVALID), (dict(pos=None), INVALID), (dict(stride=-1), INVALID),
    (dict(q=desc([1026, 1, 1, 1])), UNSUPPORTED), (dict(q=desc([0, 4, 10, 2]), n_dims=2), INVALID), (dict(q=desc([64, 1, 1 << 20, 1 << 12])), INVALID),
    (dict(q=desc([64, 4, 10, 2], nb={0: 8})), INVALID), (dict(q_dst=desc([64, 4, 10, 1])), INVALID), (dict(q_dst=None), INVALID),
    (dict(q_dst=desc([64, 4, 10, 2], GB + 256)), INVALID), (dict(q_dst=desc([64, 4, 10, 2], 9 * GB - 64)), INVALID),      # over the input; over the weights
    (dict(k=desc([64, 2, 10, 2], 4 * GB), k_dst=None), INVALID), (dict(k=desc([32, 2, 10, 2], 4 * GB)), INVALID),
    (dict(q=desc([64, 0, 10, 2]), k=desc([64, 2, 10, 2], 4 * GB)), INVALID),
])
def test_qk_refusals(kw, status):
    assert qk(**kw) == status, L.stx_last_error()
    assert L.stx_last_error()


@pytest.mark.parametrize("change", [
    dict(dy=None), dict(dy=desc([64, 4, 9, 2], 2 * GB)), dict(q=None), dict(dk=desc([64, 2, 10, 2], 5 * GB)), dict(dw_k=GB * 12), dict(dq=desc([64, 4, 9, 2], 4 * GB)),
    dict(dq=desc([64, 4, 10, 2], GB + 256)), dict(dq=desc([64, 4, 10, 2], 2 * GB + 256)), dict(dw_q=GB + 64), dict(ws=None), dict(ws=GB * 16 + 64), dict(nbytes=16),
    dict(ws=GB - 256), dict(eps=-1.0), dict(type=3), dict(pos=None), dict(dq=desc([64, 4, 10, 2], 9 * GB - 64)),
])
def test_qk_back_refusals(change):
    p = dict(dy=desc([64, 4, 10, 2], 2 * GB), q=desc([64, 4, 10, 2]), dq=desc([64, 4, 10, 2], 4 * GB), dk=None, dw_q=GB * 10, dw_k=None, ws=GB * 16, nbytes=1 << 20,
             eps=1e-6, type=F32, pos=GB * 8, **{})
    p.update(change)
    if "ws" in change and change["ws"] == GB - 256:
        p["nbytes"] = 1 << 30
    r = stx.rope_params(64)
    rc = L.stx_qk_norm_rope_back(ref(p["dy"]), None, ref(p["q"]), None, p["type"], p["pos"], 0, ctypes.byref(r), GB * 9, None, 0, p["eps"], ref(p["dq"]),
                                 ref(p["dk"]), p["dw_q"], p["dw_k"], p["ws"], p["nbytes"], None)
    assert rc == INVALID and L.stx_last_error()


def test_qk_workspace_size():
    size = L.stx_qk_norm_rope_back_workspace_size
    q = desc([64, 4, 10, 2])
    assert size(ref(q), None, F32, 64, 0) == 20 * 2 * 64 * 4 and size(ref(q), None, F32, 64, 1) == 20 * 4 * 64 * 4
    assert size(ref(desc([64, 4, 0, 2])), None, F32, 64, 0) == 0
    for bad in ((None, None, F32, 64, 0), (ref(q), None, 9, 64, 0), (ref(q), None, F32, 63, 0), (ref(q), None, F32, 66, 0), (ref(desc([2048, 1])), None, F32, 64, 0)):
        assert size(*bad) == 0


# ------------------------------------------------------------------ softmax with a position bias
REL = dict(x=desc([50, 20, 4, 2], GB), dst=desc([50, 20, 4, 2], 2 * GB), type=F32, table=GB * 5, scale=1.0, buckets=(32, 128, True, False), size=None)
REL_BAD = [
    (dict(type=5), INVALID), (dict(x=None), INVALID), (dict(x=desc([50, 20, 4, 2], GB, nb={0: 8})), INVALID), (dict(dst=None), INVALID),
    (dict(dst=desc([50, 20, 4, 1], 2 * GB)), INVALID), (dict(dst=desc([50, 20, 4, 2], GB + 200)), INVALID), (dict(dst=desc([50, 20, 4, 2], GB * 5 - 64)), INVALID),
    (dict(table=None), INVALID), (dict(scale=float("inf")), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(buckets=(1, 128, False, False)), INVALID), (dict(buckets=(2, 128, True, False)), INVALID), (dict(buckets=(33, 128, True, False)), INVALID),
    (dict(buckets=(32, 8, True, False)), INVALID), (dict(buckets=(32, 16, False, False)), INVALID), (dict(buckets=(0, 8, False, False)), INVALID),
    (dict(buckets=(512, 2000, True, False)), UNSUPPORTED), (dict(buckets=(32, 2049, True, False)), UNSUPPORTED), (dict(size=8), INVALID),
    (dict(x=desc([8, 8, 1 << 16, 2], GB), dst=desc([8, 8, 1 << 16, 2], 8 * GB)), INVALID),
    (dict(dst=desc([50, 20, 4, 2], 2 * GB, nb={1: 0})), INVALID), (dict(dst=desc([50, 20, 4, 2], 2 * GB, nb={1: 100})), INVALID),
]


def rel_of(p):
    r = stx.rel_params(*p["buckets"])
    if p["size"] is not None:
        r.size = p["size"]
    return r


@pytest.mark.parametrize("change,status", REL_BAD)
def test_rel_refusals(change, status):
    p = {**REL, **change}
    rc = L.stx_soft_max_rel(ref(p["x"]), p["type"], p["table"], ctypes.byref(rel_of(p)), p["scale"], None, None, ref(p["dst"]), None)
    assert rc == status and L.stx_last_error()


@pytest.mark.parametrize("change,status", [c for c in REL_BAD if "table" not in c[0] and "dst" not in c[0]] + [
    (dict(dy=None), INVALID), (dict(dy=desc([50, 20, 4, 1], 3 * GB)), INVALID), (dict(dst=desc([50, 20, 4, 2], GB)), INVALID),        # dx over y
    (dict(dst=desc([50, 20, 4, 2], 3 * GB)), INVALID), (dict(ws=None), INVALID), (dict(ws=GB * 16 + 8), INVALID), (dict(nbytes=64), INVALID),
    (dict(table=GB * 16), INVALID), (dict(lengths=GB * 16), INVALID)])
def test_rel_back_refusals(change, status):
    p = {**REL, "dy": desc([50, 20, 4, 2], 3 * GB), "ws": GB * 16, "nbytes": 1 << 30, "lengths": None, **change}
    if "x" in change and change["x"] is not None and change["x"].ne[2] == 1 << 16:
        p["dy"], p["dst"] = desc(list(change["x"].ne), 30 * GB), desc(list(change["x"].ne), 40 * GB)
    rc = L.stx_soft_max_rel_back(ref(p["dy"]), ref(p["x"]), p["type"], ctypes.byref(rel_of(p)), p["scale"], p["lengths"], None, ref(p["dst"]), p["table"],
                                 p["ws"], p["nbytes"], None)
    assert rc == status and L.stx_last_error()


def test_rel_workspace_size():
    size = L.stx_soft_max_rel_back_workspace_size
    assert size(ref(desc([50, 20, 4, 2])), BF16, 32) > 0 and size(ref(desc([50, 0, 4, 2])), F32, 32) == 0
    for bad in ((None, F32, 32), (ref(desc([50, 20])), 5, 32), (ref(desc([50, 20])), F32, 0), (ref(desc([50, 20])), F32, 257), (ref(desc([-1, 20])), F32, 32)):
        assert size(*bad) == 0


# ------------------------------------------------------------------------ differential attention
def diff(back=False, type=F32, **change):
    s = SIZE.get(type, 4)
    p = dict(q=desc([64, 8, 10, 2], GB, type), k=desc([64, 4, 30, 2], 2 * GB, type), v=desc([128, 2, 30, 2], 3 * GB, type), out=desc([128, 4, 10, 2], 4 * GB, type),
             second=desc([128, 4, 10, 2], 5 * GB, type), lse=6 * GB, lam=7 * GB, scale=0.125, lengths=None, ws=64 * GB, nbytes=1 << 34, dy=desc([128, 4, 10, 2], 8 * GB, type),
             dq=desc([64, 8, 10, 2], 9 * GB, type), dk=desc([64, 4, 30, 2], 10 * GB, type), dv=desc([128, 2, 30, 2], 11 * GB, type), dlam=12 * GB)
    assert s
    p.update(change)
    r = {n: ref(p[n]) for n in ("q", "k", "v", "out", "second", "dy", "dq", "dk", "dv")}
    if back:
        return L.stx_diff_attention_back(r["dy"], r["q"], r["k"], r["v"], type, p["lam"], p["scale"], 0, p["lengths"], None, r["out"], r["second"], p["lse"], r["dq"],
                                         r["dk"], r["dv"], p["dlam"], p["ws"], p["nbytes"], None)
    return L.stx_diff_attention(r["q"], r["k"], r["v"], type, p["lam"], p["scale"], 0, p["lengths"], None, r["out"], r["second"], p["lse"], p["ws"], p["nbytes"], None)


SHAPES = [
    (dict(type=9), INVALID), (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(lam=None), INVALID),
    (dict(q=desc([64, 7, 10, 2], GB)), INVALID), (dict(k=desc([64, 3, 30, 2], 2 * GB)), INVALID), (dict(k=desc([32, 4, 30, 2], 2 * GB)), INVALID),
    (dict(k=desc([64, 4, 30, 1], 2 * GB)), INVALID), (dict(v=desc([128, 3, 30, 2], 3 * GB)), INVALID), (dict(v=desc([128, 2, 29, 2], 3 * GB)), INVALID),
    (dict(k=desc([64, 6, 30, 2], 2 * GB), v=desc([128, 3, 30, 2], 3 * GB)), INVALID),                       # 4 heads on 3
    (dict(q=desc([64, 0, 10, 2], GB)), INVALID), (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(q=desc([130, 8, 10, 2], GB), k=desc([130, 4, 30, 2], 2 * GB)), UNSUPPORTED), (dict(v=desc([257, 2, 30, 2], 3 * GB)), UNSUPPORTED),
    (dict(q=desc([64, 8, 10, 2], GB, nb={0: 8})), INVALID), (dict(out=None), INVALID), (dict(out=desc([127, 4, 10, 2], 4 * GB)), INVALID),
    (dict(second=desc([128, 4, 9, 2], 5 * GB)), INVALID), (dict(ws=None), INVALID), (dict(ws=64 * GB + 16), INVALID), (dict(nbytes=100), INVALID),
]


@pytest.mark.parametrize("change,status", SHAPES + [
    (dict(out=desc([128, 4, 10, 2], GB)), INVALID), (dict(out=desc([128, 4, 10, 2], 3 * GB + 512)), INVALID), (dict(second=desc([128, 4, 10, 2], 4 * GB)), INVALID),
    (dict(out=desc([128, 4, 10, 2], 4 * GB, nb={1: 256})), INVALID), (dict(lse=GB), INVALID), (dict(lse=7 * GB), INVALID), (dict(out=desc([128, 4, 10, 2], 64 * GB)), INVALID)])
def test_diff_refusals(change, status):
    if "ws" in change or "nbytes" in change or any(v is not None and isinstance(v, stx.Tensor) and v.data == 64 * GB for v in change.values()):
        change = {**change, "k": desc([64, 4, 30000, 2], 20 * GB), "v": desc([128, 2, 30000, 2], 30 * GB)}     # a call that splits its keys
    assert diff(**change) == status, L.stx_last_error()
    assert L.stx_last_error()


@pytest.mark.parametrize("change,status", SHAPES + [
    (dict(dy=None), INVALID), (dict(dy=desc([128, 4, 9, 2], 8 * GB)), INVALID), (dict(second=None), INVALID), (dict(lse=None), INVALID),
    (dict(dk=None), INVALID), (dict(dv=None), INVALID), (dict(dq=desc([64, 8, 9, 2], 9 * GB)), INVALID), (dict(dk=desc([64, 4, 29, 2], 10 * GB)), INVALID),
    (dict(dq=desc([64, 8, 10, 2], GB)), INVALID), (dict(dv=desc([128, 2, 30, 2], 10 * GB)), INVALID), (dict(dlam=7 * GB), INVALID), (dict(dlam=64 * GB), INVALID),
    (dict(dq=desc([64, 8, 10, 2], 9 * GB, nb={2: 256})), INVALID)])
def test_diff_back_refusals(change, status):
    assert diff(back=True, **change) == status, L.stx_last_error()
    assert L.stx_last_error()


def test_diff_too_many_tiles():
    many = dict(q=desc([8, 128, 1, 1 << 17], GB), k=desc([8, 128, 1, 1 << 17], 8 * GB), v=desc([8, 64, 1, 1 << 17], 16 * GB), out=desc([8, 64, 1, 1 << 17], 24 * GB),
                second=None, lse=None)
    assert diff(**many) == INVALID and b"tiles" in L.stx_last_error()


@pytest.mark.parametrize("fn", [L.stx_diff_attention_workspace_size, L.stx_diff_attention_back_workspace_size])
def test_diff_workspace_size(fn):
    q, k, v = desc([64, 8, 1, 2]), desc([64, 4, 30000, 2]), desc([128, 2, 30000, 2])
    assert fn(ref(q), ref(k), ref(v), BF16) > 0 and fn(ref(desc([64, 8, 1, 0])), ref(desc([64, 4, 3, 0])), ref(desc([128, 2, 3, 0])), F16) == 0
    for bad in ((None, ref(k), ref(v), BF16), (ref(q), None, ref(v), BF16), (ref(q), ref(k), ref(v), 9), (ref(q), ref(k), ref(desc([128, 2, 7, 2])), BF16),
                (ref(desc([64, 7, 1, 2])), ref(k), ref(v), BF16), (ref(desc([64, 8, -1, 2])), ref(k), ref(v), BF16)):
        assert fn(*bad) == 0
