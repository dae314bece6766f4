"""What is timed of the attention operators over fp32, fp16 and bf16 tensors, forward and backward:
norms of queries and keys per head with the rotation in the same pass, the softmax of scores with a
learned relative position bias by buckets, and differential attention (the difference of two softmax
maps with a learned weight).

A case names an operator ("op"), its element type and its sizes; run() is one call of it on the
buffers that a program has in hand. The sizes are those of the two transformers this library
serves: the RoFormer layers (8 heads of 64, 60 bands x 801 frames) and HTDemucs' cross-transformer
(8 heads of 64, 1,344 and 2,688 tokens), and generic ones of longer contexts. With `own` false the
operators are elementary torch products, sums and pointwise functions in 32 bits (angles and long
sums in 64); exact() restates each in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
F32, F64 = torch.float32, torch.float64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
CHUNK = 1 << 28                          # scores that the plain forms hold at a time
MOST_PAIRS = 8 * 16384 ** 2              # query-key pairs of all heads of the largest attention


def listed():
    return [
        # One new token of a streamed sequence: a call's fixed cost.
        {"name": "qk_token", "op": "qk", "type": "bf16", "batch": 1, "tokens": 1, "heads": 8, "kv_heads": 8, "dim": 64, "n_dims": 64,
         "mode": 0, "scaling": "none", "per_head": False, "packed": True, "start": 800},
        # The time axis of a RoFormer layer: q and k of 60 bands x 801 frames, out of the projection.
        {"name": "qk_time_axis", "op": "qk", "type": "f32", "batch": 60, "tokens": 801, "heads": 8, "kv_heads": 8, "dim": 64,
         "n_dims": 64, "mode": 0, "scaling": "none", "per_head": False, "packed": True, "start": 0},
        # Its training step in half precision, with weights of their own for each head.
        {"name": "qk_layer_back", "op": "qk_back", "type": "bf16", "batch": 60, "tokens": 801, "heads": 8, "kv_heads": 8, "dim": 64,
         "n_dims": 64, "mode": 0, "scaling": "none", "per_head": True, "packed": True, "start": 0},
        # The gradient of a long context past the trained one, halves layout, part of the head, shared k heads.
        {"name": "qk_long_back", "op": "qk_back", "type": "bf16", "batch": 2, "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "n_dims": 96, "mode": 2, "scaling": "yarn", "per_head": False, "packed": False, "start": 100000},
        # A batch of streamed clips, one new frame each, of different lengths.
        {"name": "rel_token", "op": "rel", "type": "bf16", "batch": 8, "heads": 8, "queries": 1, "keys": 801, "buckets": 32,
         "distance": 128, "both": False, "causal": True, "ragged": True},
        # The scores of a cross-transformer layer's tokens in full precision.
        {"name": "rel_tokens", "op": "rel", "type": "f32", "batch": 1, "heads": 8, "queries": 1344, "keys": 1344, "buckets": 32,
         "distance": 128, "both": True, "causal": False, "ragged": False},
        # The training step of clips of different lengths, padded to 801 frames (odd rows).
        {"name": "rel_frames_back", "op": "rel_back", "type": "f32", "batch": 12, "heads": 8, "queries": 801, "keys": 801, "buckets": 32,
         "distance": 128, "both": True, "causal": False, "ragged": True},
        # The training step of a long clip in half precision, buckets that reach far.
        {"name": "rel_long_back", "op": "rel_back", "type": "bf16", "batch": 1, "heads": 8, "queries": 8192, "keys": 8192, "buckets": 64,
         "distance": 1000, "both": True, "causal": False, "ragged": False},
        # Serving: one new token of eight sequences of different lengths over their caches, four heads to a cache head.
        {"name": "diff_decode", "op": "diff", "type": "bf16", "batch": 8, "queries": 1, "keys": 16384, "heads": 16, "kv_heads": 4, "dim": 64,
         "v_dim": 128, "causal": True, "ragged": True, "keep": False},
        # The time axis of a RoFormer layer (8 heads of 64 as 4 pairs), with what a training step keeps.
        {"name": "diff_time_axis", "op": "diff", "type": "bf16", "batch": 60, "queries": 801, "keys": 801, "heads": 4, "kv_heads": 4,
         "dim": 64, "v_dim": 128, "causal": False, "ragged": False, "keep": True},
        # The training step of a cross-transformer layer (one branch's tokens over the other's) in full precision.
        {"name": "diff_cross_back", "op": "diff_back", "type": "f32", "batch": 1, "queries": 1344, "keys": 2688, "heads": 4, "kv_heads": 4,
         "dim": 64, "v_dim": 128, "causal": False, "ragged": False, "keep": True},
        # The training step of a long causal context, four heads to a key head.
        {"name": "diff_long_back", "op": "diff_back", "type": "bf16", "batch": 1, "queries": 16384, "keys": 16384, "heads": 8, "kv_heads": 2,
         "dim": 64, "v_dim": 128, "causal": True, "ragged": False, "keep": True},
    ]


def log_int(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk", "qk_back", "rel", "rel_back", "diff", "diff_back"])
    c = {"op": op, "type": rng.choice(["f32", "f16", "bf16"])}
    if op.startswith("qk"):
        dim = rng.choice([32, 64, 80, 96, 128])
        kv = rng.choice([1, 2, 4, 8])
        c.update(heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, dim=dim, n_dims=rng.choice([dim, dim // 2, dim // 4 * 2 - 2]),
                 mode=rng.choice([0, 2]), scaling=rng.choice(["none", "linear", "yarn"]), per_head=rng.random() < 0.5,
                 packed=rng.random() < 0.5, start=log_int(rng, 1, 200000))
        c["batch"] = log_int(rng, 1, 64)
        most = max(1, int(5e7 / (c["batch"] * (c["heads"] + kv) * dim)))
        c["tokens"] = log_int(rng, 1, most)
    elif op.startswith("rel"):
        c.update(batch=log_int(rng, 1, 64), heads=rng.choice([1, 2, 3, 8, 16]), both=rng.random() < 0.5, ragged=rng.random() < 0.5,
                 buckets=rng.choice([8, 16, 32, 64, 128]))
        c["causal"] = rng.random() < (0.2 if c["both"] else 0.8)
        c["distance"] = log_int(rng, c["buckets"] + 1, 2000)
        most = max(16, 8 * 8192 ** 2 // (c["batch"] * c["heads"]))
        c["keys"] = log_int(rng, 2 if op == "rel_back" else 1, min(32768, most))      # over one key the gradient is 0
        c["queries"] = log_int(rng, 1, min(8192, max(1, most // c["keys"])))
    else:
        kv = rng.choice([1, 2, 4])
        dim = rng.choice([32, 40, 64, 64, 96, 128])
        c.update(heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, dim=dim, v_dim=rng.choice([dim, 2 * dim]), batch=log_int(rng, 1, 64),
                 causal=rng.random() < 0.5, ragged=rng.random() < 0.5, keep=op == "diff_back" or rng.random() < 0.5)
        # Costs no more than the largest listed case: wider heads and full precision have fewer pairs.
        most = MOST_PAIRS * 0.45 * min(1.0, 64 / dim) / (4 if c["type"] == "f32" else 1) / (c["batch"] * c["heads"])
        c["keys"] = log_int(rng, 2 if op == "diff_back" else 1, min(16384, max(16, int(most))))
        c["queries"] = log_int(rng, 1, min(16384, max(1, int(most / c["keys"]))))
    return c


# ------------------------------------------------------------------------------- inputs
class Rand:
    """Seeded device tensors."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, scale=1.0, mean=0.0, dtype=F32):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=F32).mul_(scale).add_(mean).to(dtype)


def rope_setting(c):
    """The rotation's parameters: base, scale, trained length, ramp of frequencies (YaRN)."""
    s = {"freq_base": 10000.0, "freq_scale": 1.0, "n_ctx_orig": 0, "ext_factor": 0.0, "attn_factor": 1.0, "beta_fast": 32.0,
         "beta_slow": 1.0}
    if c["scaling"] == "linear":
        s.update(freq_scale=0.25)
    elif c["scaling"] == "yarn":
        s.update(freq_base=500000.0, freq_scale=0.125, n_ctx_orig=8192, ext_factor=1.0)
    return s


def lengths_of(c):
    """Keys of each sequence: all of them, or between half and all."""
    B, N = c["batch"], c["keys"]
    return [max(1, N - (b * N) // (2 * B)) if c["ragged"] else N for b in range(B)]


def starts_of(c):
    """Position of each sequence's first query: its queries are its last tokens where there are fewer than keys."""
    return [max(0, n - c["queries"]) if c["causal"] else 0 for n in lengths_of(c)]


def pairs_of(c):
    """Query-key pairs that the masks leave, of one head."""
    total = 0
    for n, s in zip(lengths_of(c), starts_of(c)):
        if not c["causal"]:
            total += c["queries"] * n
            continue
        whole = max(0, c["queries"] - max(0, n - s))            # queries that see every key
        part = c["queries"] - whole
        total += whole * n + part * s + part * (part + 1) // 2
    return total


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c, dt, r = case, TYPES[case["type"]], Rand(seed)
    s = {"case": dict(c)}
    if c["op"].startswith("qk"):
        B, N, H, Hk, D = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        if c["packed"]:
            qkv = r.normal(B, N, H + 2 * Hk, D, scale=1.7, dtype=dt)
            s["q"], s["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hk]
        else:
            s["q"], s["k"] = r.normal(B, N, H, D, scale=1.7, dtype=dt), r.normal(B, N, Hk, D, scale=0.6, dtype=dt)
        s["pos"] = torch.arange(c["start"], c["start"] + N, device=DEV, dtype=torch.int32)
        s["setting"] = rope_setting(c)
        s["wq"] = r.normal(*((H, D) if c["per_head"] else (D,)), scale=0.2, mean=1.0)
        s["wk"] = r.normal(*((Hk, D) if c["per_head"] else (D,)), scale=0.2, mean=1.0)
        if c["op"] == "qk_back":
            s["dq"], s["dk"] = r.normal(B, N, H, D, dtype=dt), r.normal(B, N, Hk, D, dtype=dt)
        return s
    s["lengths"] = ints(lengths_of(c)) if c["ragged"] else None
    s["starts"] = ints(starts_of(c)) if c["causal"] else None
    if c["op"].startswith("rel"):
        B, H, M, N = c["batch"], c["heads"], c["queries"], c["keys"]
        s["scale"] = 0.125
        n, near, edges = bucket_edges(c)
        s["edges"] = (n, near, torch.tensor(edges, device=DEV))
        s["table"] = r.normal(c["buckets"], H, scale=0.7)
        s["x"] = r.normal(B, H, M, N, scale=12.0, dtype=dt)
        if c["op"] == "rel_back":
            s["y"] = plain_rel(s).to(dt)                        # what the forward pass left
            del s["x"]
            s["dy"] = r.normal(B, H, M, N, dtype=dt)
        return s
    B, M, N, H, Hk, D, V = (c[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim", "v_dim"))
    s["q"], s["k"] = r.normal(B, M, 2 * H, D, dtype=dt), r.normal(B, N, 2 * Hk, D, dtype=dt)
    s["v"] = r.normal(B, N, Hk, V, dtype=dt)
    s["lam"] = r.normal(H, scale=0.15, mean=0.5)
    s["scale"] = D ** -0.5
    if c["op"] == "diff_back":
        s["out"], s["second"], s["lse"] = plain_diff(s)
        s["do"] = r.normal(B, M, H, V, dtype=dt)
    return s


# ------------------------------------------------------------------------- the plain form
def angles(pos, n_dims, freq_base, freq_scale, n_ctx_orig, ext_factor, attn_factor, beta_fast, beta_slow):
    """cos and sin [N][1][n_dims/2], scaled, in 64 bits."""
    i = torch.arange(n_dims // 2, device=pos.device, dtype=F64)
    far = torch.pow(torch.tensor(freq_base, dtype=F64, device=pos.device), -2.0 * i / n_dims)
    freq, m = freq_scale * far, attn_factor
    if ext_factor != 0.0:
        turn = lambda rot: n_dims * math.log(n_ctx_orig / (rot * 2 * math.pi)) / (2 * math.log(freq_base))  # noqa: E731
        lo, hi = max(0.0, math.floor(turn(beta_fast))), min(n_dims - 1.0, math.ceil(turn(beta_slow)))
        mix = (1.0 - ((i - lo) / max(0.001, hi - lo)).clamp(0, 1)) * ext_factor
        freq = freq * (1 - mix) + far * mix
        m = attn_factor * (1.0 + 0.1 * math.log(1.0 / freq_scale))
    theta = pos.to(F64)[:, None] * freq
    return (theta.cos() * m)[:, None], (theta.sin() * m)[:, None]


def rotate(f, cos, sin, n_dims, mode):
    rot, half = f[..., :n_dims], n_dims // 2
    if mode == 0:
        a, b = rot[..., 0::2], rot[..., 1::2]
    else:
        a, b = rot[..., :half], rot[..., half:]
    u, v = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([u, v], -1).flatten(-2) if mode == 0 else torch.cat([u, v], -1)
    return torch.cat([y, f[..., n_dims:]], -1)


def plain_qk(s):
    c = s["case"]
    cos, sin = (t.to(F32) for t in angles(s["pos"], c["n_dims"], **s["setting"]))
    out = {}
    for name in ("q", "k"):
        x, w = s[name].to(F32), s["w" + name]
        rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        if c["op"] == "qk":
            out[name] = rotate(x * rstd * w, cos, sin, c["n_dims"], c["mode"]).to(s[name].dtype)
            continue
        dz = rotate(s["d" + name].to(F32), cos, -sin, c["n_dims"], c["mode"])
        xh = x * rstd
        wdz = w * dz
        out["d" + name] = (rstd * (wdz - xh * (wdz * xh).mean(-1, keepdim=True))).to(s[name].dtype)
        out["dw" + name] = (dz * xh).sum((0, 1) if c["per_head"] else (0, 1, 2), dtype=F64).to(F32)
    return out


def bucket_edges(c):
    """Smallest distance of each bucket past the exact ones, in whole numbers: n^m >= exact^(m - k) distance^k."""
    n = c["buckets"] // 2 if c["both"] else c["buckets"]
    exact = n // 2
    m, edges = n - exact, []
    for k in range(m):
        want = exact ** (m - k) * c["distance"] ** k
        lo, hi = exact, c["distance"]
        while lo < hi:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if mid ** m >= want else (mid + 1, hi)
        edges.append(lo)
    return n, exact, edges


def buckets_of(s, rel):
    """Bucket of each key position less its query's."""
    c, n, exact, edges = s["case"], *s["edges"]
    dist = rel.abs() if c["both"] else (-rel).clamp(min=0)
    past = exact - 1 + torch.searchsorted(edges, dist, right=True)
    return torch.where(dist < exact, dist, past) + torch.where(rel > 0, n if c["both"] else 0, 0)


def seen(s, b):
    """Which keys (columns) each query (row) of sequence b sees, and the key's position less the query's."""
    c = s["case"]
    j = torch.arange(c["keys"], device=DEV)
    i = torch.arange(c["queries"], device=DEV)[:, None]
    rel = j - i - (s["starts"][b] if s["starts"] is not None else 0)
    mask = torch.ones(c["queries"], c["keys"], dtype=torch.bool, device=DEV)
    if s["lengths"] is not None:
        mask &= j < s["lengths"][b]
    if c["causal"]:
        mask &= rel <= 0
    return mask, rel


def softmax_rows(z, mask):
    """exp(z) over its row sums where mask, and the logarithm of the sums."""
    z = z.masked_fill(~mask, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    return e / total, (top + torch.log(total)).squeeze(-1)


def plain_rel(s):
    c, parts = s["case"], []
    for b in range(c["batch"]):
        mask, rel = seen(s, b)
        bias = s["table"].t()[:, buckets_of(s, rel)]                        # [H][M][N]
        parts.append(softmax_rows(s["x"][b].to(F32) * s["scale"] + bias, mask)[0].to(s["x"].dtype))
    return torch.stack(parts)


def diagonals(g):
    """Sums of [H][M][N] over equal column - row, [H][M + N - 1], from -(M - 1) on, in 64 bits."""
    H, M, N = g.shape
    wide = torch.zeros(H, M, N + M, dtype=F64, device=g.device)
    wide[:, :, :N] = g.flip(1)
    return wide.view(H, -1)[:, :M * (N + M - 1)].view(H, M, N + M - 1).sum(1)


def plain_rel_back(s):
    c, parts = s["case"], []
    H, M, N = c["heads"], c["queries"], c["keys"]
    table = torch.zeros(H, c["buckets"], dtype=F64, device=DEV)
    for b in range(c["batch"]):
        mask, _ = seen(s, b)
        # In 64 bits: a row's terms add up to 0, and where most of its keys share a bucket so does that bucket's sum.
        y, dy = s["y"][b].to(F64), s["dy"][b].to(F64)
        g = torch.where(mask, y * (dy - (y * dy).sum(-1, keepdim=True)), 0.0)
        parts.append((s["scale"] * g).to(s["y"].dtype))
        rel = torch.arange(N + M - 1, device=DEV) - (M - 1) - (s["starts"][b] if s["starts"] is not None else 0)
        hot = (buckets_of(s, rel)[:, None] == torch.arange(c["buckets"], device=DEV)).to(F64)
        table += diagonals(g) @ hot
    return {"dx": torch.stack(parts), "dtable": table.t().to(F32)}


def groups(c):
    """(sequence, first head, heads) in turns of at most CHUNK scores."""
    per = max(1, min(c["heads"], CHUNK // (c["queries"] * c["keys"])))
    return [(b, h, min(per, c["heads"] - h)) for b in range(c["batch"]) for h in range(0, c["heads"], per)]


def of_heads(s, b, h, n):
    """q1, q2, k1, k2 [n][tokens][D] and v [n][keys][V] of heads h to h + n - 1 in 32 bits; shared ones repeated."""
    c = s["case"]
    head = torch.arange(h, h + n, device=DEV)
    kv = torch.div(head, c["heads"] // c["kv_heads"], rounding_mode="floor")
    rows = lambda t, at: t[b].to(F32).transpose(0, 1)[at].contiguous()  # noqa: E731
    return rows(s["q"], 2 * head), rows(s["q"], 2 * head + 1), rows(s["k"], 2 * kv), rows(s["k"], 2 * kv + 1), rows(s["v"], kv)


def plain_diff(s):
    c, dt = s["case"], s["q"].dtype
    B, M, H, V = c["batch"], c["queries"], c["heads"], c["v_dim"]
    out, second = (torch.empty(B, M, H, V, dtype=dt, device=DEV) for _ in range(2))
    lse = torch.empty(B, H, 2, M, dtype=F32, device=DEV)
    if c["batch"] * H * M * c["keys"] <= CHUNK:
        return plain_diff_whole(s)
    for b, h, n in groups(c):
        q1, q2, k1, k2, v = of_heads(s, b, h, n)
        mask, _ = seen(s, b)
        o = []
        for m, (q, k) in enumerate(((q1, k1), (q2, k2))):
            p, lse[b, h:h + n, m] = softmax_rows(torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"], mask)
            o.append(torch.matmul(p, v))
        lam = s["lam"][h:h + n, None, None]
        out[b, :, h:h + n] = (o[0] - lam * o[1]).transpose(0, 1)
        second[b, :, h:h + n] = o[1].transpose(0, 1)
    return out, second, lse


def masks_whole(s):
    """seen() of all sequences, [B][1][M][N]."""
    c = s["case"]
    j = torch.arange(c["keys"], device=DEV)
    mask = torch.ones(1, 1, c["queries"], c["keys"], dtype=torch.bool, device=DEV)
    if s["lengths"] is not None:
        mask = mask & (j < s["lengths"][:, None, None, None])
    if c["causal"]:
        mask = mask & (j <= torch.arange(c["queries"], device=DEV)[:, None] + s["starts"][:, None, None, None])
    return mask


def maps_whole(s):
    """q, k [2][B][H][tokens][D], v [B][H][keys][V] in 32 bits, and both maps and their sums' logarithms."""
    c = s["case"]
    B, M, N, H, Hk, D = (c[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    q = s["q"].to(F32).view(B, M, H, 2, D).permute(3, 0, 2, 1, 4).contiguous()
    k = s["k"].to(F32).view(B, N, Hk, 2, D).permute(3, 0, 2, 1, 4).repeat_interleave(H // Hk, 2).contiguous()
    v = s["v"].to(F32).permute(0, 2, 1, 3).repeat_interleave(H // Hk, 1).contiguous()
    p, lse = softmax_rows(torch.matmul(q, k.transpose(3, 4).contiguous()) * s["scale"], masks_whole(s))
    return q, k, v, p, lse


def plain_diff_whole(s):
    _, _, v, p, lse = maps_whole(s)
    o1, o2 = torch.matmul(p[0], v), torch.matmul(p[1], v)
    out = o1 - s["lam"][:, None, None] * o2
    dt = s["q"].dtype
    return out.transpose(1, 2).to(dt).contiguous(), o2.transpose(1, 2).to(dt).contiguous(), lse.permute(1, 2, 0, 3).contiguous()


def plain_diff_back(s):
    c, dt = s["case"], s["q"].dtype
    M, N, H, Hk = c["queries"], c["keys"], c["heads"], c["kv_heads"]
    dq = torch.empty_like(s["q"])
    dk, dv = torch.zeros_like(s["k"], dtype=F32), torch.zeros_like(s["v"], dtype=F32)
    dlam = torch.zeros(H, dtype=F64, device=DEV)
    if c["batch"] * H * M * N <= CHUNK:
        return plain_diff_back_whole(s)
    for b, h, n in groups(c):
        q1, q2, k1, k2, v = of_heads(s, b, h, n)
        mask, _ = seen(s, b)
        do = s["do"][b].to(F32).transpose(0, 1)[h:h + n].contiguous()
        o2 = s["second"][b].to(F32).transpose(0, 1)[h:h + n]
        lam = s["lam"][h:h + n, None, None]
        o1 = s["out"][b].to(F32).transpose(0, 1)[h:h + n] + lam * o2
        dp = torch.matmul(do, v.transpose(1, 2).contiguous())
        mix = 0.0
        for m, (q, k, o, f) in enumerate(((q1, k1, o1, 1.0), (q2, k2, o2, -lam))):
            z = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
            p = torch.exp(z - s["lse"][b, h:h + n, m, :, None]).masked_fill(~mask, 0.0)
            mix = mix + f * p
            if m == 1:
                dlam[h:h + n] -= (p * dp).sum((1, 2), dtype=F64)
            ds = f * p * (dp - (do * o).sum(-1, keepdim=True)) * s["scale"]
            dq[b, :, 2 * h + m:2 * (h + n):2] = torch.matmul(ds, k).transpose(0, 1)
            part = torch.matmul(ds.transpose(1, 2).contiguous(), q)
            for i in range(n):
                dk[b, :, (h + i) // (H // Hk) * 2 + m] += part[i]
        part = torch.matmul(mix.transpose(1, 2).contiguous(), do)
        for i in range(n):
            dv[b, :, (h + i) // (H // Hk)] += part[i]
    return {"dq": dq, "dk": dk.to(dt), "dv": dv.to(dt), "dlam": dlam.to(F32)}


def plain_diff_back_whole(s):
    c, dt = s["case"], s["q"].dtype
    B, M, N, H, Hk, D = (c[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    q, k, v, _, _ = maps_whole(s)
    lse = s["lse"].permute(2, 0, 1, 3)[..., None]
    p = torch.exp(torch.matmul(q, k.transpose(3, 4).contiguous()) * s["scale"] - lse).masked_fill(~masks_whole(s), 0.0)
    do, o2 = (s[n].to(F32).transpose(1, 2).contiguous() for n in ("do", "second"))
    lam = s["lam"][:, None, None]
    o1 = s["out"].to(F32).transpose(1, 2) + lam * o2
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    dots = torch.stack([(do * o1).sum(-1, keepdim=True), (do * o2).sum(-1, keepdim=True)])
    f = torch.stack([torch.ones_like(lam), -lam])[:, None]
    ds = f * p * (dp - dots) * s["scale"]
    dq = torch.matmul(ds, k).permute(1, 3, 2, 0, 4).reshape(B, M, 2 * H, D)
    dk = torch.matmul(ds.transpose(3, 4).contiguous(), q).view(2, B, Hk, H // Hk, N, D).sum(3).permute(1, 3, 2, 0, 4).reshape(B, N, 2 * Hk, D)
    dv = torch.matmul((p[0] - lam * p[1]).transpose(2, 3).contiguous(), do).view(B, Hk, H // Hk, N, -1).sum(2).transpose(1, 2)
    return {"dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt).contiguous(), "dlam": -(p[1] * dp).sum((0, 2, 3), dtype=F64).to(F32)}


def plain(s):
    c, op = s["case"], s["case"]["op"]
    if op.startswith("qk"):
        return plain_qk(s)
    if op == "rel":
        return {"y": plain_rel(s)}
    if op == "rel_back":
        return plain_rel_back(s)
    if op == "diff":
        out, second, lse = plain_diff(s)
        return {"out": out, "second": second, "lse": lse} if c["keep"] else {"out": out}
    return plain_diff_back(s)


# ---------------------------------------------------------------- the framework's operators
def library():
    path = os.path.join(os.getcwd(), "stems.cpp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import stx
    return stx


def called(s):
    stx = library()
    c, op = s["case"], s["case"]["op"]
    if op.startswith("qk"):
        params = stx.rope_params(c["n_dims"], c["mode"], **s["setting"])
        if op == "qk":
            q, k = stx.qk_norm_rope(s["q"], s["pos"], params, s["wq"], s["k"], s["wk"], eps=EPS)
            return {"q": q, "k": k}
        dq, dwq, dk, dwk = stx.qk_norm_rope_back(s["dq"], s["q"], s["pos"], params, s["wq"], s["dk"], s["k"], s["wk"], eps=EPS)
        return {"dq": dq, "dwq": dwq, "dk": dk, "dwk": dwk}
    if op.startswith("rel"):
        params = stx.rel_params(c["buckets"], c["distance"], bidirectional=c["both"], causal=c["causal"])
        if op == "rel":
            return {"y": stx.soft_max_rel(s["x"], s["table"], params, s["scale"], s["lengths"], s["starts"])}
        dx, dtable = stx.soft_max_rel_back(s["dy"], s["y"], params, s["scale"], s["lengths"], s["starts"])
        return {"dx": dx, "dtable": dtable}
    mask = dict(scale=s["scale"], causal=c["causal"], lengths=s["lengths"], starts=s["starts"])
    if op == "diff":
        out, second, lse = stx.diff_attention(s["q"], s["k"], s["v"], s["lam"], keep=c["keep"], **mask)
        return {"out": out, "second": second, "lse": lse} if c["keep"] else {"out": out}
    dq, dk, dv, dlam = stx.diff_attention_back(s["do"], s["q"], s["k"], s["v"], s["lam"], s["out"], s["second"], s["lse"], **mask)
    return {"dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def run(state):
    if own:
        return called(state)
    return plain(state)


def work(case):
    c, size, back = case, BYTES[case["type"]], case["op"].endswith("_back")
    if c["op"].startswith("qk"):
        rows = c["batch"] * c["tokens"] * (c["heads"] + c["kv_heads"])
        weights = 4 * c["dim"] * (c["heads"] + c["kv_heads"] if c["per_head"] else 2)
        return {"bytes": (3 if back else 2) * rows * c["dim"] * size + 4 * c["tokens"] + (2 if back else 1) * weights,
                "flops": rows * ((13 if back else 4) * c["dim"] + 3 * c["n_dims"])}
    pairs = pairs_of(c) * c["heads"]
    extra = 4 * c["batch"] * (c["ragged"] + c["causal"])
    if c["op"].startswith("rel"):
        whole = c["batch"] * c["heads"] * c["queries"] * c["keys"]
        return {"bytes": size * ((2 if back else 1) * pairs + whole) + 4 * c["buckets"] * c["heads"] + extra,
                "flops": (6 if back else 5) * pairs}
    queries, keys, D, V = c["batch"] * c["queries"], sum(lengths_of(c)), c["dim"], c["v_dim"]
    q, kv, o = queries * 2 * c["heads"] * D, keys * c["kv_heads"] * (2 * D + V), queries * c["heads"] * V
    kept = 4 * queries * 2 * c["heads"] + size * o              # both maps' sums, and the second's output
    if back:
        all_kv = c["batch"] * c["keys"] * c["kv_heads"] * (2 * D + V)
        return {"bytes": size * (2 * q + kv + all_kv + 2 * o) + kept + 8 * c["heads"] + extra, "flops": pairs * (12 * D + 4 * V)}
    return {"bytes": size * (q + kv + o) + (kept if c["keep"] else 0) + 4 * c["heads"] + extra,
            "flops": pairs * (4 * D + 4 * V)}


# ------------------------------------------------------------------------ the definitions
def exact_qk(c, s):
    half, t = c["n_dims"] // 2, s["setting"]
    turn = torch.empty(half, dtype=F64)
    for i in range(half):
        f = t["freq_base"] ** (-2.0 * i / c["n_dims"])
        if t["ext_factor"] != 0.0:
            edge = [c["n_dims"] * math.log(t["n_ctx_orig"] / (2 * math.pi * b)) / (2 * math.log(t["freq_base"]))
                    for b in (t["beta_fast"], t["beta_slow"])]
            lo, hi = max(0, math.floor(edge[0])), min(c["n_dims"] - 1, math.ceil(edge[1]))
            far = t["ext_factor"] * (1.0 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo))))
            f = f * far + t["freq_scale"] * f * (1.0 - far)
        else:
            f *= t["freq_scale"]
        turn[i] = f
    m = t["attn_factor"] * (1.0 - 0.1 * math.log(t["freq_scale"]) if t["ext_factor"] != 0.0 else 1.0)
    pos = s["pos"].to(F64)
    z = torch.polar(torch.full((pos.numel(), half), m, dtype=F64, device=DEV), pos[:, None] * turn.to(DEV))[:, None]
    first = slice(0, c["n_dims"], 2) if c["mode"] == 0 else slice(0, half)
    second = slice(1, c["n_dims"], 2) if c["mode"] == 0 else slice(half, c["n_dims"])

    def turned(x, z):
        y = x.clone()
        w = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z
        y[..., first], y[..., second] = w.real, w.imag
        return y

    out = {}
    for name in ("q", "k"):
        x, w = s[name].to(F64), s["w" + name].to(F64)
        norm = (x.square().sum(-1, keepdim=True) / c["dim"] + EPS).sqrt()
        if c["op"] == "qk":
            out[name] = turned(w * x / norm, z)
        else:
            dz = turned(s["d" + name].to(F64), z.conj())
            out["d" + name] = w * dz / norm - x * (w * dz * x).sum(-1, keepdim=True) / (c["dim"] * norm ** 3)
            dw = (dz * x / norm).sum((0, 1))
            out["dw" + name] = dw if c["per_head"] else dw.sum(0)
    return out


def exact_bias(c, s, b):
    """bias [H][M][N] and bucket [M][N] of sequence b, the latter from logarithms in 64 bits."""
    at = torch.arange(c["queries"], device=DEV, dtype=F64)[:, None] + float(starts_of(c)[b])
    rel = torch.arange(c["keys"], device=DEV, dtype=F64) - at
    n = c["buckets"] // 2 if c["both"] else c["buckets"]
    near = n // 2
    d = rel.abs() if c["both"] else torch.relu(-rel)
    # A distance on a border gives a whole number, which the logarithms may miss by their rounding.
    steps = torch.floor(torch.log(d.clamp(min=near) / near) * ((n - near) / math.log(c["distance"] / near)) + 1e-11)
    index = torch.where(d < near, d, near + torch.minimum(steps, torch.full_like(steps, n - near - 1)))
    index = (index + (rel > 0) * (n if c["both"] else 0)).long()
    hide = torch.zeros(c["queries"], c["keys"], dtype=torch.bool, device=DEV)
    hide[:, lengths_of(c)[b]:] = True
    if c["causal"]:
        hide |= rel > 0
    return s["table"].to(F64).t()[:, index], index, hide


def exact_rel(c, s):
    if c["op"] == "rel":
        y = torch.empty(s["x"].shape, dtype=F64, device=DEV)
        for b in range(c["batch"]):
            bias, _, hide = exact_bias(c, s, b)
            z = s["x"][b].to(F64) * s["scale"] + bias
            z[:, hide] = -math.inf
            y[b] = torch.softmax(z, -1)
        return {"y": y}
    dx = torch.zeros(s["y"].shape, dtype=F64, device=DEV)
    table = torch.zeros(c["buckets"], c["heads"], dtype=F64, device=DEV)
    for b in range(c["batch"]):
        _, index, hide = exact_bias(c, s, b)
        for h in range(c["heads"]):
            y, dy = s["y"][b, h].to(F64), s["dy"][b, h].to(F64).masked_fill(hide, 0.0)
            g = y * dy - y * (y * dy).sum(-1, keepdim=True)
            g[hide] = 0.0
            dx[b, h] = g * s["scale"]
            order = torch.argsort(index.flatten()) if index.numel() < 1 << 20 else None
            if order is not None:
                sums = torch.cat([torch.zeros(1, dtype=F64, device=DEV), g.flatten()[order].cumsum(0)])
                ends = torch.cumsum(torch.bincount(index.flatten(), minlength=c["buckets"]), 0)
                table[:, h] += torch.diff(sums[ends], prepend=sums[:1])
            else:
                for k in range(c["buckets"]):
                    table[k, h] += torch.where(index == k, g, 0.0).sum()
    return {"dx": dx, "dtable": table}


def exact_diff(c, s):
    B, M, N, H, Hk = (c[n] for n in ("batch", "queries", "keys", "heads", "kv_heads"))
    if c["op"] == "diff":
        out, second = (torch.empty(B, M, H, c["v_dim"], dtype=F64, device=DEV) for _ in range(2))
        lse = torch.empty(B, H, 2, M, dtype=F64, device=DEV)
    else:
        dq, dk, dv = (torch.zeros(s[n].shape, dtype=F64, device=DEV) for n in ("q", "k", "v"))
        dlam = torch.zeros(H, dtype=F64, device=DEV)
    for b, (n, start) in enumerate(zip(lengths_of(c), starts_of(c))):
        hide = None
        if c["causal"]:
            hide = torch.arange(n, device=DEV) > torch.arange(start, start + M, device=DEV)[:, None]
        for h in range(H):
            g, lam = h // (H // Hk), float(s["lam"][h])
            v = s["v"][b, :n, g].to(F64)
            p = []
            for m in range(2):
                z = torch.mm(s["q"][b, :, 2 * h + m].to(F64), s["k"][b, :n, 2 * g + m].to(F64).t().contiguous()) * s["scale"]
                if hide is not None:
                    z[hide] = -math.inf
                if c["op"] == "diff":
                    lse[b, h, m] = torch.logsumexp(z, -1)
                p.append(torch.softmax(z, -1))
                del z
            if c["op"] == "diff":
                second[b, :, h] = torch.mm(p[1], v)
                out[b, :, h] = torch.mm(p[0] - lam * p[1], v)
                continue
            do = s["do"][b, :, h].to(F64)
            dmap = torch.mm(do, v.t().contiguous())
            dv[b, :n, g] += torch.mm((p[0] - lam * p[1]).t().contiguous(), do)
            dlam[h] -= (p[1] * dmap).sum()
            for m, weight in ((0, 1.0), (1, -lam)):
                dz = p[m] * (dmap - (p[m] * dmap).sum(-1, keepdim=True)) * (weight * s["scale"])
                dq[b, :, 2 * h + m] = torch.mm(dz, s["k"][b, :n, 2 * g + m].to(F64))
                dk[b, :n, 2 * g + m] += torch.mm(dz.t().contiguous(), s["q"][b, :, 2 * h + m].to(F64))
                del dz
    if c["op"] == "diff":
        return {"out": out, "second": second, "lse": lse} if c["keep"] else {"out": out}
    return {"dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("qk"):
        return exact_qk(case, s)
    if case["op"].startswith("rel"):
        return exact_rel(case, s)
    return exact_diff(case, s)
