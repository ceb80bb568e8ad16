"""A paged cache of keys and values in few bits and the attention over it, as timed cases.

  store    rows of K and V go into their pages, quantised, and the same rows come back (axhip_kv_write, axhip_kv_read)
  load     whole sequences come back from their pages (axhip_kv_read)
  step     one or a few new tokens of each sequence over its pages (axhip_attn_paged)
  chunk    chunks of prompts, and single tokens beside them, over their pages (axhip_attn_paged)

A cache holds rows of heads in 16 bits (f16), 8 (i8) or 4 (mx4).  Device buffers that a program hands to the C ABI are torch tensors here.  Everything runs on
the null stream.
"""
import ctypes as C
import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = ("f16", "i8", "mx4")
BITS = {"f16": 16, "i8": 8, "mx4": 4}
_lib = {}


def _hip():
    """The library, loaded and initialised once per process."""
    if not _lib:
        from axiom_amd.hip import AxHip, KvCache, KvRules
        _lib["cache"], _lib["rules"] = KvCache, KvRules
        _lib["hip"] = AxHip()
        _lib["hip"].init()
    return _lib["hip"]


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # serving: a step writes one token of each of 16 sequences
        {"name": "store_step_16_i8", "kind": "store", "type": "i8", "batch": 16, "new": 1, "steps": 0, "seq": 2000, "kv": 8, "dim": 128, "page": 16},
        # serving: five prompts of unlike lengths arrive together
        {"name": "store_prompts_4096_mx4", "kind": "store", "type": "mx4", "batch": 5, "new": 4096, "steps": 0, "seq": 4096, "kv": 8, "dim": 128, "page": 64},
        # sequences brought back for a pass over contiguous rows, small heads
        {"name": "load_6x1000_i8", "kind": "load", "type": "i8", "batch": 6, "new": 0, "steps": 0, "seq": 1000, "kv": 4, "dim": 64, "page": 16},
        # the same for long sequences, odd heads in 16 bits
        {"name": "load_8x8192_f16", "kind": "load", "type": "f16", "batch": 8, "new": 0, "steps": 0, "seq": 8192, "kv": 8, "dim": 80, "page": 128},
        # one sequence, one token, a short cache: latency
        {"name": "step_1x500_i8", "kind": "step", "type": "i8", "batch": 1, "new": 1, "steps": 0, "seq": 500, "heads": 16, "kv": 4, "dim": 64, "page": 16,
         "window": 0, "sinks": 0, "cap": 0.0, "slopes": False},
        # a batch of ragged sequences over a large cache, small pages: bandwidth
        {"name": "step_32x4096_i8", "kind": "step", "type": "i8", "batch": 32, "new": 1, "steps": 0, "seq": 4096, "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "window": 0, "sinks": 0, "cap": 50.0, "slopes": False},
        # long sequences of which a window and the first tokens are seen, biased by distance
        {"name": "step_window_16x16384_f16", "kind": "step", "type": "f16", "batch": 16, "new": 1, "steps": 0, "seq": 16384, "heads": 16, "kv": 4, "dim": 64, "page": 64,
         "window": 2048, "sinks": 4, "cap": 0.0, "slopes": True},
        # two tokens at once (one of them a guess) over very long sequences in 4 bits
        {"name": "step_8x32768_mx4", "kind": "step", "type": "mx4", "batch": 8, "new": 2, "steps": 0, "seq": 32768, "heads": 64, "kv": 8, "dim": 128, "page": 64,
         "window": 0, "sinks": 0, "cap": 0.0, "slopes": False},
        # a short turn of a conversation behind a long one
        {"name": "chunk_1x64_over_8192_i8", "kind": "chunk", "type": "i8", "batch": 1, "new": 64, "steps": 0, "seq": 8192, "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "window": 0, "sinks": 0, "cap": 0.0, "slopes": False},
        # a server's batch: four chunks of prompts and twenty sequences that get one token, heads between the usual sizes, capped scores
        {"name": "chunk_mixed_24x3000_f16", "kind": "chunk", "type": "f16", "batch": 24, "new": 600, "steps": 20, "seq": 3000, "heads": 16, "kv": 4, "dim": 80, "page": 32,
         "window": 0, "sinks": 0, "cap": 50.0, "slopes": False},
        # whole prompts under a window, every head with keys of its own, 4 bits
        {"name": "chunk_window_4x4096_mx4", "kind": "chunk", "type": "mx4", "batch": 4, "new": 4096, "steps": 0, "seq": 4096, "heads": 16, "kv": 16, "dim": 64, "page": 64,
         "window": 1024, "sinks": 4, "cap": 0.0, "slopes": False},
        # large chunks over what came before them: the most arithmetic of all
        {"name": "chunk_2x2048_over_4096_i8", "kind": "chunk", "type": "i8", "batch": 2, "new": 2048, "steps": 0, "seq": 4096, "heads": 32, "kv": 8, "dim": 128, "page": 64,
         "window": 0, "sinks": 0, "cap": 0.0, "slopes": False},
    ]


def _size(rng, lo, hi, grain):
    """Log-uniform in [lo, hi]; half of the draws on the grid of `grain` (sizes that models choose), half anywhere (sizes that data gives)."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    if rng.random() < 0.5:
        v = round(v / grain) * grain
    return int(min(hi, max(lo, round(v))))


def draw(rng):
    kind = rng.choice(["store", "load", "step", "step", "chunk", "chunk"])
    kv = rng.choice([1, 2, 4, 8])
    c = {"kind": kind, "type": rng.choice(TYPES), "steps": 0, "kv": kv, "dim": rng.choice([32, 40, 64, 64, 80, 96, 112, 128, 128]), "page": rng.choice([16, 32, 64, 128, 256])}
    if kind in ("store", "load"):
        rows = _size(rng, 1, 16000, 16)
        c["batch"] = max(1, min(_size(rng, 1, 32, 1), rows))
        if kind == "store":
            c["new"] = max(1, rows // c["batch"])
            c["seq"] = c["new"] if c["new"] > 1 else _size(rng, 1, 4000, 16)
        else:
            c["new"], c["seq"] = 0, max(1, rows // c["batch"])
        return c
    heads = kv * rng.choice([1, 2, 4, 8])
    c.update(heads=heads, window=rng.choice([0, 0, 128, 1000, 4096]), cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.25)
    c["sinks"] = rng.choice([0, 1, 4]) if c["window"] else 0
    if kind == "step":
        c["seq"] = _size(rng, 1, 32768, 64)
        c["new"] = min(c["seq"], rng.choice([1, 1, 1, 2, 4]))
        # at most the cache of the largest listed step
        c["batch"] = max(1, min(_size(rng, 1, 64, 1), 8 * 32768 * 8 * 128 // (c["seq"] * kv * c["dim"])))
        return c
    c["new"] = _size(rng, 1, 4096, 32)
    c["seq"] = _size(rng, c["new"], 8192, 64)
    # at most the scores of the largest listed chunk
    most = 2 * 2048 * 4096 * 32
    while c["new"] * c["seq"] * heads > most:
        c["seq"] = max(c["new"], c["seq"] // 2)
        c["new"] = min(c["new"], max(1, most // (c["seq"] * heads)))
    chunks = max(1, min(_size(rng, 1, 8, 1), most // (c["new"] * c["seq"] * heads)))
    c["steps"] = rng.choice([0, 0, 3, 16])
    c["batch"] = chunks + c["steps"]
    return c


def _shape(c):
    """New tokens and lengths of the sequences: those of the case, whatever the seed."""
    rng = random.Random("%d %d %d %d" % (c["batch"], c["new"], c["steps"], c["seq"]))
    b, n, seq, chunks = c["batch"], c["new"], c["seq"], c["batch"] - c["steps"]
    if c["kind"] == "load":
        lens = [rng.randint((seq + 1) // 2, seq) for _ in range(b - 1)] + [seq]
        return lens, lens
    if c["kind"] == "step" or n == 1:
        new = [n] * b
    else:
        new = [n] + [rng.randint((n + 1) // 2, n) for _ in range(chunks - 1)] + [1] * c["steps"]
    if c["kind"] == "store" and n > 1:
        return new, new                                   # prompts that arrive
    lens = [rng.randint(max(k, seq // 2), max(k, seq)) for k in new]
    lens[0] = max(new[0], seq)
    order = list(range(b))
    rng.shuffle(order)
    return [new[i] for i in order], [lens[i] for i in order]


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 31)
    return g


def _normal(g, shape):
    return torch.empty(shape, device=DEV).normal_(0.0, 1.0, generator=g)


def _row_bytes(c):
    return (c["dim"] * BITS[c["type"]] // 8 + 15) // 16 * 16


def prepare(case, seed):
    g, rng = _generator(seed), random.Random(seed * 31 + 11)
    c = case
    b, kv, d, page = c["batch"], c["kv"], c["dim"], c["page"]
    new, lens = _shape(c)
    cols = (max(lens) + page - 1) // page + 1
    used = [(n + page - 1) // page for n in lens]
    pages = sum(used) + 3
    order = list(range(pages))
    rng.shuffle(order)
    table = []
    for n in used:                                        # pages as they were free; behind a sequence's last there is none
        table.append([order.pop() for _ in range(n)] + [-1] * (cols - n))
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    s = {"case": c, "new": new, "lens_host": lens, "rows": first[-1], "pages": pages,
         "table": torch.tensor(table, device=DEV, dtype=torch.int32), "first": torch.tensor(first, device=DEV, dtype=torch.int32),
         "lens": torch.tensor(lens, device=DEV, dtype=torch.int32)}
    size = _row_bytes(c)
    for x in "kv":
        s[x + "_pages"] = torch.zeros((pages, kv, page, size), device=DEV, dtype=torch.uint8)
        s[x + "_scale"] = torch.zeros((pages, kv, page, 4), device=DEV, dtype=torch.uint8)
    if c["kind"] == "store":
        # a row of the fused projection behind its query heads: keys, values
        s["kv_rows"] = _normal(g, (s["rows"], 2 * kv * d))
    else:                                                 # sequences that were written before
        total = sum(lens)
        at = torch.tensor([0] + lens, device=DEV).cumsum(0)
        pos = torch.arange(total, device=DEV) - at[:-1].repeat_interleave(s["lens"])
        seq = torch.arange(b, device=DEV).repeat_interleave(s["lens"])
        for x in "kv":
            _put(s, x, _normal(g, (total, kv, d)), seq, pos)
    if c["kind"] in ("store", "load"):
        s["k_out"], s["v_out"] = (torch.empty((s["rows"], kv * d), device=DEV) for _ in range(2))
    else:
        h = c["heads"]
        s["q"], s["o"] = _normal(g, (s["rows"], h * d)), torch.empty((s["rows"], h * d), device=DEV)
        s["lse"] = torch.empty((s["rows"], h), device=DEV)
        s["scale"] = 1 / math.sqrt(d)
        s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, h + 1, device=DEV, dtype=torch.float64) / h)).float() if c["slopes"] else None
    return s


# ---- the plain form --------------------------------------------------------------------------------------------------

def _quantised(c, x):
    """x [rows, heads, dim] as bytes of payload [rows, heads, row bytes] and of scales [rows, heads, 4]"""
    rows, heads, d = x.shape
    out = torch.zeros((rows, heads, _row_bytes(c)), device=DEV, dtype=torch.uint8)
    if c["type"] == "mx4":
        groups = (d + 31) // 32
        y = torch.zeros((rows, heads, groups * 32), device=DEV)
        y[..., :d] = x
        y = y.view(rows, heads, groups, 32)
        e = (torch.frexp(y.abs().amax(-1))[1] - 3).clamp_min(-127)          # top = m 2^ex, 1/2 <= m < 1
        v = torch.ldexp(y, -e[..., None]).abs()
        v = torch.where(v < 2, torch.round(v * 2) / 2, torch.where(v < 4, torch.round(v), 2 * torch.round(v / 2))).clamp_max(6)
        code = torch.where(v < 2, v * 2, torch.where(v < 4, v + 2, v / 2 + 4)).to(torch.uint8) + 8 * (y < 0).to(torch.uint8)
        code = code.view(rows, heads, groups * 32)
        out[..., :groups * 16] = code[..., 0::2] + 16 * code[..., 1::2]
        scale = torch.zeros((rows, heads, 4), device=DEV, dtype=torch.uint8)
        scale[..., :groups] = (e + 127).to(torch.uint8)
        return out, scale
    top = x.abs().amax(-1)
    if c["type"] == "f16":
        scale = torch.ldexp(torch.ones_like(top), (torch.frexp(top)[1] - 15).clamp_min(-100))
        out[..., :2 * d] = (x / scale[..., None]).half().view(torch.uint8)
    else:
        scale = (top.double() / 127).float()
        n = torch.round(x.double() / scale.double()[..., None]).clamp(-127, 127)
        out[..., :d] = torch.where(scale[..., None] > 0, n, 0.0).to(torch.int8).view(torch.uint8)
    return out, scale[..., None].contiguous().view(torch.uint8)


def _place(s, seq, pos):
    c = s["case"]
    return s["table"][seq, pos // c["page"]].long(), pos % c["page"]


def _put(s, x, rows, seq, pos):
    payload, scale = _quantised(s["case"], rows)
    page, row = _place(s, seq, pos)
    s[x + "_pages"][page, :, row] = payload
    s[x + "_scale"][page, :, row] = scale


def _get(s, x, seq, pos):
    """Rows [.., heads, dim] in 32 bits at positions `pos` of sequences `seq`"""
    c = s["case"]
    d = c["dim"]
    page, row = _place(s, seq, pos)
    payload, scale = s[x + "_pages"][page.clamp_min(0), :, row], s[x + "_scale"][page.clamp_min(0), :, row]
    if c["type"] == "mx4":
        groups = (d + 31) // 32
        ladder = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
        code = torch.stack([payload & 15, payload >> 4], -1).flatten(-2)[..., :groups * 32].int()
        v = ladder[code & 7] * (1 - 2 * (code >> 3))
        e = scale[..., :groups].int() - 127
        return torch.ldexp(v.unflatten(-1, (groups, 32)), e[..., None]).flatten(-2)[..., :d]
    held = payload[..., :2 * d].contiguous().view(torch.float16) if c["type"] == "f16" else payload[..., :d].view(torch.int8)
    return held.float() * scale.contiguous().view(torch.float32)


def _new_rows(s):
    """Sequences and positions of the new rows"""
    n = s["first"].diff()
    seq = torch.arange(s["case"]["batch"], device=DEV).repeat_interleave(n, output_size=s["rows"])
    return seq, torch.arange(s["rows"], device=DEV) - s["first"][1:][seq] + s["lens"][seq]


def _attend(s, q, seqs, lens, longest):
    """q [b, n, heads, dim] of sequences `seqs` [b] -> o [b, n, heads * dim], lse [b, n, heads]"""
    c = s["case"]
    b, n, h, d = q.shape
    kv, g = c["kv"], h // c["kv"]
    j = torch.arange(longest, device=DEV)
    k, v = (_get(s, x, seqs[:, None], j[None].expand(b, -1)).transpose(1, 2).contiguous() for x in "kv")       # [b, kv, keys, dim]
    q = q.view(b, n, kv, g, d).permute(0, 2, 3, 1, 4).reshape(b, kv, g * n, d)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    x = x.view(b, h, n, longest)
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    p = lens[:, None] - n + torch.arange(n, device=DEV)                     # [b, n]
    back = p[..., None] - j
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * back.float()[:, None]
    seen = back >= 0
    if c["window"]:
        seen = seen & ((back < c["window"]) | (j < c["sinks"]))
    x = x.masked_fill(~seen[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul((e / total).view(b, kv, g * n, longest), torch.where((j < lens[:, None])[:, None, :, None], v, 0.0))
    o = o.view(b, h, n, d).transpose(1, 2).reshape(b, n, h * d)
    return o, (top + total.log())[..., 0].transpose(1, 2)


def _plain(s):
    c = s["case"]
    kv, d = c["kv"], c["dim"]
    if c["kind"] in ("store", "load"):
        seq, pos = _new_rows(s)
        if c["kind"] == "store":
            for i, x in enumerate("kv"):
                _put(s, x, s["kv_rows"][:, i * kv * d:(i + 1) * kv * d].view(-1, kv, d), seq, pos)
        return {x: _get(s, x, seq, pos).reshape(-1, kv * d) for x in "kv"}
    q = s["q"].view(s["rows"], c["heads"], d)
    if c["kind"] == "step":
        o, lse = _attend(s, q.view(c["batch"], c["new"], c["heads"], d), torch.arange(c["batch"], device=DEV), s["lens"], max(s["lens_host"]))
        return {"o": o.flatten(0, 1), "lse": lse.flatten(0, 1)}
    o, lse, at = [], [], 0
    for i, (n, length) in enumerate(zip(s["new"], s["lens_host"])):
        a, b = _attend(s, q[None, at:at + n], torch.arange(i, i + 1, device=DEV), s["lens"][i:i + 1], length)
        o.append(a[0])
        lse.append(b[0])
        at += n
    return {"o": torch.cat(o), "lse": torch.cat(lse)}


# ---- one pass --------------------------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(s):
    hip, c = _hip(), s["case"]
    L, kv, d = hip.L, c["kv"], c["dim"]
    cache = C.byref(_lib["cache"](type=TYPES.index(c["type"]), page_rows=c["page"], pages=s["pages"], heads=kv, dk=d, k=_ptr(s["k_pages"]), v=_ptr(s["v_pages"]),
                                  k_scale=_ptr(s["k_scale"]), v_scale=_ptr(s["v_scale"]), table=_ptr(s["table"]), table_ld=s["table"].shape[1]))
    b, rows, most, uniform = c["batch"], s["rows"], max(s["new"]), c["kind"] == "step" or len(set(s["new"])) == 1
    first = None if uniform else _ptr(s["first"])
    if c["kind"] in ("store", "load"):
        if c["kind"] == "store":
            x = s["kv_rows"].data_ptr()
            hip.check(L.axhip_kv_write(cache, x, 2 * kv * d, x + 4 * kv * d, 2 * kv * d, first, _ptr(s["lens"]), b, rows, most))
        hip.check(L.axhip_kv_read(cache, _ptr(s["k_out"]), kv * d, _ptr(s["v_out"]), kv * d, first, _ptr(s["lens"]), b, rows, most))
        return {"k": s["k_out"], "v": s["v_out"]}
    h = c["heads"]
    rules = C.byref(_lib["rules"](cap=c["cap"], window=c["window"], sinks=c["sinks"], slopes=_ptr(s["slopes"])))
    hip.check(L.axhip_attn_paged(_ptr(s["q"]), h * d, cache, _ptr(s["o"]), h * d, _ptr(s["lse"]), first, _ptr(s["lens"]), b, rows, h, most, max(s["lens_host"]), s["scale"], rules))
    return {"o": s["o"], "lse": s["lse"]}


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    c = case
    new, lens = _shape(c)
    held = 2 * c["kv"] * (c["dim"] * BITS[c["type"]] / 8 + 4)              # of a position: keys and values
    wide = 2 * c["kv"] * c["dim"] * 4
    if c["kind"] == "store":
        return {"bytes": int(sum(new) * 2 * (wide + held)), "flops": int(sum(new) * wide)}
    if c["kind"] == "load":
        return {"bytes": int(sum(new) * (wide + held)), "flops": int(sum(new) * wide // 4)}
    pairs = keys = 0
    for n, length in zip(new, lens):
        for_window = c["window"] or length
        low = max(0, length - n - for_window + 1)                          # the first key in the first query's window
        keys += length - low + min(c["sinks"], low)
        for p in range(length - n, length):
            begin = max(0, p - for_window + 1)
            pairs += p + 1 - begin + min(c["sinks"], begin)
    return {"bytes": int(keys * held + sum(new) * c["heads"] * (2 * c["dim"] + 1) * 4), "flops": int(4 * pairs * c["heads"] * c["dim"])}


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------------

def _rounded(c, x):
    """What the cache holds for rows x [.., dim] of 64-bit numbers"""
    if c["type"] == "f16":
        top = x.abs().amax(-1, keepdim=True)
        s = 2.0 ** torch.floor(torch.log2(top)) * 2.0 ** -14              # tops are far from powers of two or are ones
        y = x / s
        step = (2.0 ** (torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -14))) - 10)).clamp_min(2.0 ** -24)
        return torch.round(y / step) * step * s
    if c["type"] == "i8":
        s = (x.abs().amax(-1, keepdim=True) / 127).float().double()
        return torch.round(x / s) * s
    out = torch.zeros_like(x)
    steps = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV, dtype=torch.float64)
    for at in range(0, c["dim"], 32):
        part = x[..., at:at + 32]
        s = 2.0 ** (torch.floor(torch.log2(part.abs().amax(-1, keepdim=True))) - 2)
        y = (part / s).abs()
        up = torch.searchsorted(steps, y.contiguous()).clamp(1, 7)         # the neighbours' ladder: steps[up - 1] < y <= steps[up], or past the last
        low, high = steps[up - 1], steps[up]
        to_high = (y - low > high - y) | ((y - low == high - y) & (up % 2 == 0))
        out[..., at:at + 32] = torch.where(to_high, high, low) * part.sign() * s
    return out


def _held(s, x, i, length):
    """Sequence i's rows [length, heads, dim] in 64 bits, page by page, from the bytes that the cache holds"""
    c = s["case"]
    d, size = c["dim"], c["page"]
    parts = []
    for at in range(0, length, size):
        page = int(s["table"][i, at // size])
        n = min(size, length - at)
        raw, scale = s[x + "_pages"][page, :, :n], s[x + "_scale"][page, :, :n]
        if c["type"] == "f16":
            y = raw.contiguous().view(torch.float16)[..., :d].double() * scale.contiguous().view(torch.float32).double()
        elif c["type"] == "i8":
            y = raw.contiguous().view(torch.int8)[..., :d].double() * scale.contiguous().view(torch.float32).double()
        else:
            y = torch.empty((c["kv"], n, 2 * raw.shape[-1]), device=DEV, dtype=torch.float64)
            for half, code in enumerate((raw % 16, raw // 16)):
                low = (code % 8).double()                                  # two bits of exponent, one of mantissa
                e, m = torch.floor(low / 2), low % 2
                v = torch.where(e > 0, (1 + m / 2) * 2.0 ** (e - 1), m / 2)
                y[..., half::2] = torch.where(code >= 8, -v, v)
            y = y[..., :d] * (2.0 ** (scale.double() - 127)).repeat_interleave(32, -1)[..., :d]
        parts.append(y.transpose(0, 1))
    return torch.cat(parts)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kv, d = c["kv"], c["dim"]
    if c["kind"] == "store":
        k, v = s["kv_rows"].double().view(-1, 2, kv, d).unbind(1)
        return {"k": _rounded(c, k).reshape(-1, kv * d), "v": _rounded(c, v).reshape(-1, kv * d)}
    if c["kind"] == "load":
        return {x: torch.cat([_held(s, x, i, n) for i, n in enumerate(s["lens_host"])]).reshape(-1, kv * d) for x in "kv"}
    h = c["heads"]
    q = s["q"].double().view(-1, h, d)
    o, lse = torch.zeros((s["rows"], h, d), device=DEV, dtype=torch.float64), torch.zeros((s["rows"], h), device=DEV, dtype=torch.float64)
    at = 0
    for i, (n, length) in enumerate(zip(s["new"], s["lens_host"])):
        k, v = _held(s, "k", i, length), _held(s, "v", i, length)
        p = torch.arange(length - n, length, device=DEV)[:, None]
        j = torch.arange(length, device=DEV)[None]
        seen = j <= p
        if c["window"]:
            seen = seen & ((j > p - c["window"]) | (j < c["sinks"]))
        for m in range(h):
            x = q[at:at + n, m] @ k[:, m * kv // h].T * s["scale"]
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if s["slopes"] is not None:
                x = x - s["slopes"][m].double() * (p - j)
            x = torch.where(seen, x, -math.inf)
            total = torch.logsumexp(x, -1)
            lse[at:at + n, m] = total
            o[at:at + n, m] = torch.exp(x - total[:, None]) @ v[:, m * kv // h]
        at += n
    return {"o": o.reshape(s["rows"], h * d), "lse": lse}
