"""The operators between an attention layer's projections, as timed cases.

Four kinds of call, each on rows that hold heads side by side, as a fused projection writes them:

  rope     rotation of heads by their position, forward and backward (axhip_rope_rows)
  qknorm   root-mean-square norm of each query and key head and its rotation in one pass, forward and backward
           (axhip_qk_norm_rope_fwd, axhip_qk_norm_rope_bwd)
  attend   attention whose scores are capped by a tanh, biased by distance, or masked by documents, by a prefix or by lengths,
           with keys and values shared by groups of query heads, forward and backward (axhip_attn_fwd, axhip_attn_bwd)
  step     the same forward for one or a few new tokens of each sequence over a cache (axhip_attn_fwd)

Device buffers that a program hands to the C ABI are torch tensors here.  Everything runs on the null stream.
"""
import ctypes as C
import math
import random

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
_lib = {}


def _hip():
    """The library, loaded and initialised once per process."""
    if not _lib:
        from axiom_amd.hip import AttnRules, AxHip
        _lib["rules"] = AttnRules
        _lib["hip"] = AxHip()
        _lib["hip"].init()
    return _lib["hip"]


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # serving: one token of each of 8 sequences that have come far, interleaved pairs, keys and queries in one call
        {"name": "rope_step_8", "kind": "rope", "rows": 8, "heads": 20, "dim": 64, "rot": 64, "layout": 0, "far": 1000000, "amplitude": 1.0, "grad": False},
        # training: the gradient of a batch of long prompts, half layout on part of the head, amplitude of a context that was stretched
        {"name": "rope_grad_16000", "kind": "rope", "rows": 16000, "heads": 24, "dim": 128, "rot": 96, "layout": 1, "far": 8000, "amplitude": 1.1, "grad": True},
        # serving: a step of 16 sequences
        {"name": "qknorm_step_16", "kind": "qknorm", "rows": 16, "heads": 16, "kv": 4, "dim": 64, "rot": 64, "layout": 1, "far": 100000, "amplitude": 1.0, "grad": False},
        # prompts, large heads, keys shared by four query heads
        {"name": "qknorm_8192", "kind": "qknorm", "rows": 8192, "heads": 32, "kv": 8, "dim": 128, "rot": 128, "layout": 1, "far": 8192, "amplitude": 1.0, "grad": False},
        # training: the gradient for eight ragged sequences of 500, heads of an odd size, part of each rotated
        {"name": "qknorm_grad_4000", "kind": "qknorm", "rows": 4000, "heads": 16, "kv": 16, "dim": 80, "rot": 40, "layout": 0, "far": 500, "amplitude": 1.0, "grad": True},
        # a prompt of a decoder with capped scores, keys shared by four query heads
        {"name": "attend_capped_4x1024x128", "kind": "attend", "batch": 4, "seq": 1024, "heads": 16, "kv": 4, "dim": 128, "cap": 50.0, "slopes": False, "causal": True,
         "prefix": False, "lens": False, "docs": 0, "grad": False},
        # pretraining: documents packed to one long row, most of the square masked
        {"name": "attend_docs_1x8192x64", "kind": "attend", "batch": 1, "seq": 8192, "heads": 16, "kv": 16, "dim": 64, "cap": 0.0, "slopes": False, "causal": True,
         "prefix": False, "lens": False, "docs": 12, "grad": False},
        # a padded batch with a bias by distance, ragged length, heads between the kernels' own sizes
        {"name": "attend_distance_3x777x80", "kind": "attend", "batch": 3, "seq": 777, "heads": 12, "kv": 12, "dim": 80, "cap": 0.0, "slopes": True, "causal": True,
         "prefix": False, "lens": True, "docs": 0, "grad": False},
        # fine-tuning: short sequences whose prompts are seen from everywhere
        {"name": "attend_grad_prefix_8x512x64", "kind": "attend", "batch": 8, "seq": 512, "heads": 8, "kv": 8, "dim": 64, "cap": 0.0, "slopes": False, "causal": True,
         "prefix": True, "lens": True, "docs": 0, "grad": True},
        # training: capped scores on long rows, keys shared by two query heads, the largest of all
        {"name": "attend_grad_capped_2x2048x128", "kind": "attend", "batch": 2, "seq": 2048, "heads": 16, "kv": 8, "dim": 128, "cap": 30.0, "slopes": False, "causal": True,
         "prefix": False, "lens": False, "docs": 0, "grad": True},
        # serving: one sequence, one token, a short cache: latency
        {"name": "step_1x500x64", "kind": "step", "batch": 1, "new": 1, "seq": 500, "room": 1024, "heads": 16, "kv": 4, "dim": 64, "cap": 0.0, "slopes": True},
        # serving: a batch of ragged sequences over a large cache: bandwidth
        {"name": "step_32x4096x128", "kind": "step", "batch": 32, "new": 1, "seq": 4096, "room": 4100, "heads": 32, "kv": 8, "dim": 128, "cap": 50.0, "slopes": False},
    ]


def _size(rng, lo, hi, grain):
    """Log-uniform in [lo, hi]; half of the draws on the grid of `grain` (sizes that models choose), half anywhere (sizes that data gives)."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    if rng.random() < 0.5:
        v = round(v / grain) * grain
    return int(min(hi, max(lo, round(v))))


def draw(rng):
    kind = rng.choice(["rope", "qknorm", "attend", "attend", "step"])
    dim = rng.choice([32, 48, 64, 80, 96, 112, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4])
    if kind in ("rope", "qknorm"):
        c = {"kind": kind, "rows": _size(rng, 1, 16000, 16), "heads": heads, "kv": kv, "dim": dim, "rot": rng.choice([dim, dim, dim // 2, dim // 4]),
             "layout": rng.randrange(2), "far": _size(rng, 100, 1000000, 100), "amplitude": rng.choice([1.0, 1.2]), "grad": rng.random() < 0.5}
        if kind == "rope":
            del c["kv"]
        return c
    if kind == "attend":
        grad = rng.random() < 0.5
        # at most the largest listed case's scores
        most = (1 if grad else 2) * 2048 * 2048 * 32
        seq = min(_size(rng, 1, 4096, 32), math.isqrt(most // heads))
        batch = max(1, min(_size(rng, 1, 16, 1), most // (seq * seq * heads)))
        causal = rng.random() < 0.75
        return {"kind": kind, "batch": batch, "seq": seq, "heads": heads, "kv": kv, "dim": dim, "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "slopes": rng.random() < 0.3,
                "causal": causal, "prefix": causal and rng.random() < 0.3, "lens": rng.random() < 0.4, "docs": rng.choice([0, 0, 2, 7]) if seq >= 32 else 0, "grad": grad}
    seq = _size(rng, 1, 16384, 64)
    batch = max(1, min(_size(rng, 1, 64, 1), 32 * 4096 * 8 * 128 // (seq * kv * dim)))
    return {"kind": kind, "batch": batch, "new": min(seq, rng.choice([1, 1, 1, 2, 5])), "seq": seq, "room": seq + _size(rng, 1, 100, 16), "heads": heads, "kv": kv, "dim": dim,
            "cap": rng.choice([0.0, 50.0]), "slopes": rng.random() < 0.3}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 29)
    return g


def _normal(g, shape, std=1.0, mean=0.0):
    return torch.empty(shape, device=DEV).normal_(mean, std, generator=g)


def _documents(rng, seq, n, pad):
    """Ids of n packed documents of unlike lengths, then -1 for `pad` rows."""
    cuts = sorted(rng.sample(range(1, seq - pad), min(n, seq - pad) - 1)) if n > 1 else []
    ids, at = [], 0
    for d, end in enumerate(cuts + [seq - pad]):
        ids += [d] * (end - at)
        at = end
    return ids + [-1] * pad


def prepare(case, seed):
    g, rng = _generator(seed), random.Random(seed * 31 + 7)
    c, kind = case, case["kind"]
    s = {"case": c, "scale": 1 / math.sqrt(c["dim"])}
    if kind in ("rope", "qknorm"):
        rows, d, rot = c["rows"], c["dim"], c["rot"]
        heads = c["heads"] + c.get("kv", 0)
        s["pos"] = torch.randint(0, c["far"], (rows,), device=DEV, generator=g, dtype=torch.int32)
        s["freq"] = (10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)).float()
        if kind == "rope":
            s["x"], s["y"] = _normal(g, (rows, heads * d)), torch.empty((rows, heads * d), device=DEV)
            return s
        # a row of the fused projection: query heads, key heads, value heads
        s["x"] = _normal(g, (rows, (heads + c["kv"]) * d), 2.0)
        s["gq"], s["gk"] = _normal(g, (d,), 0.2, 1.0), _normal(g, (d,), 0.2, 1.0)
        s["inv"] = torch.empty((rows, heads), device=DEV)
        if c["grad"]:
            s["dy"] = _normal(g, (rows, heads * d))
            s["dx"], s["dgq"], s["dgk"] = torch.empty((rows, heads * d), device=DEV), torch.empty(d, device=DEV), torch.empty(d, device=DEV)
            s["inv"] = (s["x"][:, :heads * d].view(rows, heads, d).square().mean(-1) + EPS).rsqrt()
        else:
            s["y"] = torch.empty((rows, heads * d), device=DEV)
        return s
    b, n, h, kv, d = c["batch"], c["seq"], c["heads"], c["kv"], c["dim"]
    s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, h + 1, device=DEV, dtype=torch.float64) / h)).float() if c["slopes"] else None
    s["prefix"] = s["lens"] = s["start"] = s["docs"] = None
    if kind == "step":
        new = c["new"]
        lens = [rng.randint(max(new, n // 2), n) for _ in range(b)]
        lens[rng.randrange(b)] = n
        s["lens"] = torch.tensor(lens, device=DEV, dtype=torch.int32)
        s["start"] = s["lens"] - new                      # the new tokens are the last of each sequence
        s["q"] = _normal(g, (b, new, h, d))
        s["k"], s["v"] = _normal(g, (b, c["room"], kv, d)), _normal(g, (b, c["room"], kv, d))
        s["o"], s["lse"] = torch.empty((b, new, h * d), device=DEV), torch.empty((b, h, new), device=DEV)
        return s
    # the fused projection [b, n, q | k | v]
    s["qkv"] = _normal(g, (b, n, (h + 2 * kv) * d))
    if c["lens"]:
        s["lens"] = torch.tensor([rng.randint((n + 1) // 2, n) for _ in range(b)], device=DEV, dtype=torch.int32)
    if c["prefix"]:
        s["prefix"] = torch.tensor([rng.randint(0, n // 2) for _ in range(b)], device=DEV, dtype=torch.int32)
    if c["docs"]:
        s["docs"] = torch.tensor([_documents(rng, n, c["docs"], rng.randint(0, n // 8)) for _ in range(b)], device=DEV, dtype=torch.int32)
    s["o"], s["lse"] = torch.empty((b, n, h * d), device=DEV), torch.empty((b, h, n), device=DEV)
    if c["grad"]:
        o, lse = _attend(s)                               # what the forward pass left
        s["o"].copy_(o)
        s["lse"].copy_(lse)
        s["do"] = _normal(g, (b, n, h * d))
        s["dqkv"] = torch.empty_like(s["qkv"])
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------

def _turn(s, x, back):
    """x [rows, heads, dim] turned by its rows' angles (back: by their opposites, the transpose)."""
    c = s["case"]
    rot = c["rot"]
    angle = s["pos"].double()[:, None] * s["freq"].double()
    cos, sin = ((f(angle) * c["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    if back:
        sin = -sin
    out = x.clone()
    if c["layout"] == 0:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    return out


def _gammas(s):
    """[heads of queries and keys, dim]"""
    c = s["case"]
    return torch.cat([s["gq"].expand(c["heads"], -1), s["gk"].expand(c["kv"], -1)])


def _qknorm(s):
    c = s["case"]
    rows, d, heads = c["rows"], c["dim"], c["heads"] + c["kv"]
    x = s["x"][:, :heads * d].view(rows, heads, d)
    if not c["grad"]:
        inv = (x.square().mean(-1) + EPS).rsqrt()
        y = _turn(s, x * inv[..., None] * _gammas(s), False)
        return {"y": y.view(rows, heads * d), "inv": inv}
    dn = _turn(s, s["dy"].view(rows, heads, d), True)
    hat = x * s["inv"][..., None]
    dg = (dn * hat).sum(0, dtype=torch.float64)
    dh = dn * _gammas(s)
    dx = (dh - hat * (dh * hat).mean(-1, keepdim=True)) * s["inv"][..., None]
    return {"dx": dx.view(rows, heads * d), "dgq": dg[:c["heads"]].sum(0).float(), "dgk": dg[c["heads"]:].sum(0).float()}


def _heads(s):
    """Queries, and keys and values repeated for every query head: [b, heads, rows, dim]; positions of the queries [b, rows], keys' count and indices."""
    c = s["case"]
    h, kv, d = c["heads"], c["kv"], c["dim"]
    if c["kind"] == "step":
        q, k, v = s["q"], s["k"][:, :c["seq"]], s["v"][:, :c["seq"]]
    else:
        b, n = c["batch"], c["seq"]
        q, k, v = (x.view(b, n, -1, d) for x in s["qkv"].split((h * d, kv * d, kv * d), -1))
    q = q.transpose(1, 2).contiguous()
    k, v = (x.transpose(1, 2).repeat_interleave(h // kv, 1) for x in (k, v))
    start = s["start"][:, None] if s["start"] is not None else torch.zeros((c["batch"], 1), device=DEV, dtype=torch.int32)
    p = start + torch.arange(q.shape[2], device=DEV, dtype=torch.int32)
    return q, k, v, p


def _seen(s, p, nk):
    """[b, 1, rows, keys]: which keys a query sees."""
    c = s["case"]
    j = torch.arange(nk, device=DEV, dtype=torch.int32)
    end = s["lens"] if s["lens"] is not None else torch.full((c["batch"],), nk, device=DEV, dtype=torch.int32)
    ok = (j < end[:, None])[:, None, :].expand(-1, p.shape[1], -1)
    if c.get("causal", True):
        before = j <= p[..., None]
        if s["prefix"] is not None:
            before = before | (j < s["prefix"][:, None])[:, None, :]
        ok = ok & before & (p < end[:, None])[..., None]
    if s["docs"] is not None:
        ok = ok & (s["docs"][:, :, None] == s["docs"][:, None, :]) & (s["docs"] >= 0)[:, :, None]
    return ok[:, None]


def _scores(s, q, k, p):
    """Scores before the mask, and the derivative of the cap (None without one)."""
    c = s["case"]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    slope = None
    if c["cap"]:
        t = torch.tanh(x / c["cap"])
        x, slope = t * c["cap"], 1 - t * t
    if s["slopes"] is not None:
        j = torch.arange(k.shape[2], device=DEV, dtype=torch.int32)
        x = x - s["slopes"][:, None, None] * (p[..., None] - j).abs().float()[:, None]
    return x, slope


def _attend(s):
    c = s["case"]
    q, k, v, p = _heads(s)
    x, _ = _scores(s, q, k, p)
    x = x.masked_fill(~_seen(s, p, k.shape[2]), -math.inf)
    top = x.amax(-1, keepdim=True)
    e = (x - top.clamp_min(-3e38)).exp()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e / total.clamp_min(1e-30), v)
    lse = (top + total.log())[..., 0]
    return o.transpose(1, 2).reshape(c["batch"], q.shape[2], -1), lse


def _attend_grad(s):
    c = s["case"]
    b, n, h, kv, d = c["batch"], c["seq"], c["heads"], c["kv"], c["dim"]
    q, k, v, p = _heads(s)
    x, slope = _scores(s, q, k, p)
    lse = s["lse"][..., None]
    prob = torch.where(_seen(s, p, n) & (lse > -math.inf), x - lse, -math.inf).exp()
    do = s["do"].view(b, n, h, d).transpose(1, 2).contiguous()
    delta = (do * s["o"].view(b, n, h, d).transpose(1, 2)).sum(-1, keepdim=True)
    dx = prob * (torch.matmul(do, v.transpose(2, 3).contiguous()) - delta)
    if slope is not None:
        dx = dx * slope
    dx = dx * s["scale"]
    dq = torch.matmul(dx, k)
    dk = torch.matmul(dx.transpose(2, 3).contiguous(), q).view(b, kv, h // kv, n, d).sum(2)
    dv = torch.matmul(prob.transpose(2, 3).contiguous(), do).view(b, kv, h // kv, n, d).sum(2)
    return torch.cat([x.transpose(1, 2).reshape(b, n, -1) for x in (dq, dk, dv)], -1)


# ---- one pass --------------------------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _rules(s):
    c = s["case"]
    return C.byref(_lib["rules"](cap=c["cap"], causal=int(c.get("causal", True)), slopes=_ptr(s["slopes"]), prefix=_ptr(s["prefix"]), start=_ptr(s["start"]),
                                   lens=_ptr(s["lens"]), doc_q=_ptr(s["docs"]), doc_k=_ptr(s["docs"])))


def _own(s):
    hip, c = _hip(), s["case"]
    L, d, h = hip.L, c["dim"], c["heads"]
    if c["kind"] == "rope":
        hip.check(L.axhip_rope_rows(s["x"].data_ptr(), h * d, s["y"].data_ptr(), h * d, s["pos"].data_ptr(), s["freq"].data_ptr(), c["rows"], h, d, c["rot"],
                                    c["amplitude"], c["layout"], int(c["grad"])))
        return s["y"]
    kv = c["kv"]
    if c["kind"] == "qknorm":
        ld, wide = (h + kv) * d, (h + 2 * kv) * d
        if c["grad"]:
            hip.check(L.axhip_qk_norm_rope_bwd(s["dy"].data_ptr(), ld, s["x"].data_ptr(), wide, s["inv"].data_ptr(), s["dx"].data_ptr(), ld, s["gq"].data_ptr(),
                                               s["gk"].data_ptr(), s["dgq"].data_ptr(), s["dgk"].data_ptr(), s["pos"].data_ptr(), s["freq"].data_ptr(), c["rows"], h, kv, d,
                                               c["rot"], c["amplitude"], c["layout"]))
            return {"dx": s["dx"], "dgq": s["dgq"], "dgk": s["dgk"]}
        hip.check(L.axhip_qk_norm_rope_fwd(s["x"].data_ptr(), wide, s["y"].data_ptr(), ld, s["inv"].data_ptr(), s["gq"].data_ptr(), s["gk"].data_ptr(), EPS,
                                           s["pos"].data_ptr(), s["freq"].data_ptr(), c["rows"], h, kv, d, c["rot"], c["amplitude"], c["layout"]))
        return {"y": s["y"], "inv": s["inv"]}
    b, n = c["batch"], c["seq"]
    if c["kind"] == "step":
        hip.check(L.axhip_attn_fwd(s["q"].data_ptr(), h * d, s["k"].data_ptr(), kv * d, s["v"].data_ptr(), kv * d, c["room"], s["o"].data_ptr(), h * d, s["lse"].data_ptr(),
                                   b, h, kv, c["new"], n, d, s["scale"], _rules(s)))
        return s["o"], s["lse"]
    ld = (h + 2 * kv) * d
    q = s["qkv"].data_ptr()
    k = q + 4 * h * d
    v = k + 4 * kv * d
    if not c["grad"]:
        hip.check(L.axhip_attn_fwd(q, ld, k, ld, v, ld, n, s["o"].data_ptr(), h * d, s["lse"].data_ptr(), b, h, kv, n, n, d, s["scale"], _rules(s)))
        return s["o"], s["lse"]
    dq = s["dqkv"].data_ptr()
    dk = dq + 4 * h * d
    hip.check(L.axhip_attn_bwd(q, ld, k, ld, v, ld, n, s["o"].data_ptr(), h * d, s["lse"].data_ptr(), s["do"].data_ptr(), h * d, dq, ld, dk, ld, dk + 4 * kv * d, ld,
                               b, h, kv, n, n, d, s["scale"], _rules(s)))
    return s["dqkv"]


def run(s):
    if own:
        return _own(s)
    c = s["case"]
    if c["kind"] == "rope":
        return _turn(s, s["x"].view(c["rows"], c["heads"], c["dim"]), c["grad"]).view(c["rows"], -1)
    if c["kind"] == "qknorm":
        return _qknorm(s)
    if c["kind"] == "attend" and c["grad"]:
        return _attend_grad(s)
    return _attend(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "rope":
        return {"bytes": 4 * c["rows"] * (2 * c["heads"] * c["dim"] + 1), "flops": 3 * c["rows"] * c["heads"] * c["rot"]}
    if c["kind"] == "qknorm":
        heads = c["heads"] + c["kv"]
        return {"bytes": 4 * c["rows"] * ((3 if c["grad"] else 2) * heads * c["dim"] + heads + 1),
                "flops": c["rows"] * heads * ((10 if c["grad"] else 4) * c["dim"] + 3 * c["rot"])}
    b, n, h, kv, d = c["batch"], c["seq"], c["heads"], c["kv"], c["dim"]
    if c["kind"] == "step":
        keys = b * (n + (b - 1) * 0.75 * n) / b           # one sequence is full, the others between half and full
        return {"bytes": int(4 * (2 * keys * kv * d + 2 * b * c["new"] * h * d + b * c["new"] * h)), "flops": int(4 * keys * c["new"] * h * d)}
    rows = b * n
    length = 0.75 * n if c["lens"] else n                  # the keys of a sequence, between half and all of n
    queries = length if c["causal"] else n
    pairs = queries * length / 2 + (queries * length / 16 if c["prefix"] else 0) if c["causal"] else queries * length
    if c["docs"]:                                          # of n random pieces of a row two places share one with probability 2 / (n + 1)
        pairs *= 2 / (c["docs"] + 1) * 0.88
    held = rows * (h + 2 * kv) * d
    if c["grad"]:
        return {"bytes": int(4 * (2 * held + 2 * rows * h * d + rows * h)), "flops": int(10 * b * h * pairs * d)}
    return {"bytes": int(4 * (held + rows * h * d + rows * h)), "flops": int(4 * b * h * pairs * d)}


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------------

def _rotation(c, s, x, sign):
    """Pairs as complex numbers, times amplitude * e^(sign * i * angle)."""
    rot = c["rot"]
    head = x[..., :rot]
    z = torch.view_as_complex(head.unflatten(-1, (rot // 2, 2)).contiguous()) if c["layout"] == 0 else torch.complex(head[..., :rot // 2], head[..., rot // 2:])
    angle = torch.outer(s["pos"].double(), s["freq"].double())
    z = z * torch.polar(torch.full_like(angle, c["amplitude"]), sign * angle)[:, None]
    head = torch.view_as_real(z).flatten(-2) if c["layout"] == 0 else torch.cat([z.real, z.imag], -1)
    return torch.cat([head, x[..., rot:]], -1)


def _visible(c, s, i, positions, keys):
    """The keys that the queries at `positions` of sequence i see, from the rules as they are written."""
    n = int(s["lens"][i]) if s["lens"] is not None else keys
    at = torch.arange(keys, device=DEV)
    m = (at < n).expand(len(positions), keys).clone()
    if c.get("causal", True):
        shared = int(s["prefix"][i]) if s["prefix"] is not None else 0
        m &= (at[None] <= positions[:, None]) | (at[None] < shared)
        m &= (positions < n)[:, None]
    if s["docs"] is not None:
        ids = s["docs"][i]
        m &= (ids[:, None] == ids[None]) & (ids[:, None] != -1)
    return m


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "rope":
        return _rotation(c, s, s["x"].double().view(c["rows"], c["heads"], c["dim"]), -1 if c["grad"] else 1).reshape(c["rows"], -1)
    h, kv, d = c["heads"], c["kv"], c["dim"]
    if c["kind"] == "qknorm":
        rows = c["rows"]
        x = s["x"].double()[:, :(h + kv) * d].reshape(rows, h + kv, d)
        g = torch.cat([s["gq"].double().repeat(h, 1), s["gk"].double().repeat(kv, 1)])
        r = 1 / torch.sqrt((x * x).sum(-1) / d + EPS)
        if not c["grad"]:
            return {"y": _rotation(c, s, x * r[..., None] * g, 1).reshape(rows, -1), "inv": r}
        dn = _rotation(c, s, s["dy"].double().view(rows, h + kv, d), -1)
        # y = g x r, dr/dx = -r^3 x / d
        inner = (dn * g * x).sum(-1)
        dx = dn * g * r[..., None] - x * (r ** 3 * inner / d)[..., None]
        dg = torch.einsum("rhd,rhd,rh->hd", dn, x, r)
        return {"dx": dx.reshape(rows, -1), "dgq": dg[:h].sum(0), "dgk": dg[h:].sum(0)}
    b = c["batch"]
    if c["kind"] == "step":
        q, k, v = (s[x].double() for x in "qkv")
        k, v = k[:, :c["seq"]], v[:, :c["seq"]]
    else:
        q, k, v = (x.reshape(b, c["seq"], -1, d) for x in s["qkv"].double().split((h * d, kv * d, kv * d), -1))
    rows, keys, grad = q.shape[1], k.shape[1], c.get("grad", False)
    o, lse = torch.zeros((b, rows, h, d), device=DEV, dtype=torch.float64), torch.zeros((b, h, rows), device=DEV, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(b):
        first = int(s["start"][i]) if s["start"] is not None else 0
        at = torch.arange(rows, device=DEV) + first
        ok = _visible(c, s, i, at, keys)
        for m in range(h):
            kk, vv = k[i, :, m * kv // h], v[i, :, m * kv // h]
            raw = q[i, :, m] @ kk.T * s["scale"]
            x = c["cap"] * torch.tanh(raw / c["cap"]) if c["cap"] else raw
            if s["slopes"] is not None:
                x = x - s["slopes"][m].double() * (at[:, None] - torch.arange(keys, device=DEV)[None]).abs()
            x = torch.where(ok, x, -math.inf)
            lse[i, m] = torch.logsumexp(x, -1)
            prob = torch.where(ok, torch.exp(x - lse[i, m].clamp_min(-1e300)[:, None]), 0.0)
            o[i, :, m] = prob @ vv
            if grad:
                do = s["do"].double().view(b, rows, h, d)[i, :, m]
                dp = do @ vv.T
                ds = prob * (dp - (prob * dp).sum(-1, keepdim=True)) * s["scale"]
                if c["cap"]:
                    ds = ds / torch.cosh(raw / c["cap"]) ** 2
                dq[i, :, m] = ds @ kk
                dk[i, :, m * kv // h] += ds.T @ q[i, :, m]
                dv[i, :, m * kv // h] += prob.T @ do
    if grad:
        return torch.cat([x.reshape(b, rows, -1) for x in (dq, dk, dv)], -1)
    return o.reshape(b, rows, -1), lse
