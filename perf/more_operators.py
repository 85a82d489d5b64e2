"""Decoding over a paged cache: rotary positions, appending to the cache, attention over it.

A training step returns results and gradients; a serving call its result and the state it updates.  ``run`` computes the
operators in elementary torch operations (32 bits, angles in 64, rounded once at the end), or with ``own`` set calls the
package as a program does.  ``exact`` restates each in float64.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


def _rotary(name=None, **over):
    case = {"op": "rotary", "b": 1, "n": 1, "h": 16, "hk": 16, "d": 64, "rot": 64, "interleaved": False, "docs": 0,
            "start": 0, "factor": 1.0, "io": "bf16", "train": False}
    return {**({"name": name} if name else {}), **case, **over}


def _append(name=None, **over):
    case = {"op": "append", "b": 1, "n": 1, "h": 16, "hk": 16, "d": 64, "rot": 64, "interleaved": False, "ragged": False,
            "most": 1000, "page": 64, "slots_first": False, "factor": 1.0, "io": "bf16"}
    return {**({"name": name} if name else {}), **case, **over}


def _paged(name=None, **over):
    case = {"op": "attn", "b": 1, "n": 1, "h": 16, "hk": 16, "d": 64, "ragged": False, "most": 1000, "page": 64,
            "slots_first": False, "cap": 0.0, "radius": 0, "io": "bf16"}
    return {**({"name": name} if name else {}), **case, **over}


def listed():
    return [
        # Queries and keys of one new residue, serving: the smallest call, latency.
        _rotary("rotary_token_b1", start=772),
        # A training step of two rows of packed sequences, shared key heads.
        _rotary("rotary_train_b2_n4096", b=2, n=4096, h=32, hk=8, d=128, rot=128, docs=9, train=True),
        # The token attention's heads (16 of 24), part of each rotated in neighbouring pairs, odd length, fp32 training.
        _rotary("rotary_train_f32_n333", b=3, n=333, d=24, rot=16, interleaved=True, io="fp32", train=True),
        # A long prompt far behind the lengths trained on, frequencies scaled, half of the head rotated.
        _rotary("rotary_prompt_far_n16384", n=16384, h=16, hk=4, d=128, rot=64, interleaved=True, start=1000000,
                factor=32.0),
        # One new token of each of 64 sequences goes to its page.
        _append("append_token_b64", b=64, h=32, hk=8, d=128, rot=128, most=1000),
        # Four prompts of unequal length into small pages.
        _append("append_prompt_b4_n4000", b=4, n=4000, h=32, hk=8, d=128, rot=128, ragged=True, most=4300, page=16),
        # A few tokens each of three sequences, heads of 24, pages that end anywhere, fp32.
        _append("append_few_f32_b3", b=3, n=5, d=24, rot=24, interleaved=True, ragged=True, most=700, page=20,
                slots_first=True, io="fp32"),
        # One new token for each of eight sequences over long caches.
        _paged("attn_token_b8_n32768", b=8, h=32, hk=8, d=128, most=32768),
        # One new token over a short cache with the distance bias: the smallest attention call.
        _paged("attn_token_b1_n773", radius=128, most=773, page=16),
        # A full batch of sequences of moderate length, eight heads to a key head, capped scores.
        _paged("attn_token_b64_n4000", b=64, h=32, hk=4, d=128, most=4000, page=16, cap=50.0, slots_first=True),
        # A few tokens at a time, some fewer than others, fp32, pages that end inside any tile.
        _paged("attn_few_f32_b4_n5000", b=4, n=5, h=16, hk=4, ragged=True, most=5000, page=20, io="fp32"),
        # A decoding step of a layer: rotate, append, attend.
        {**_paged("step_b32_n2048", b=32, h=32, hk=8, d=128, most=2048, page=32), "op": "step", "rot": 128,
         "interleaved": False, "factor": 1.0},
    ]


def draw(rng):
    """A case of the listed ones' ranges, sizes spread over their logarithm, odd ones among them."""
    def size(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    op = rng.choice(["rotary", "append", "attn", "attn", "step"])
    h, hk = rng.choice([(16, 16), (16, 4), (8, 8), (8, 1), (32, 8), (32, 4), (7, 7)])
    d = rng.choice([24, 32, 64, 80, 128])
    io = rng.choice(["bf16", "bf16", "fp32"])
    common = {"h": h, "hk": hk, "d": d, "io": io}
    turn = {"rot": rng.choice([d, d, d // 2 // 2 * 2, 8]), "interleaved": rng.random() < 0.5,
            "factor": rng.choice([1.0, 1.0, 8.0, 32.0])}
    if op == "rotary":
        n = size(1, 16384 * 16 * 64 // ((h + hk) * d))
        return _rotary(b=rng.randint(1, 3), n=n, docs=rng.choice([0, 1 + n // 100]),
                       start=rng.choice([0, size(1, 1000000)]), train=rng.random() < 0.5, **common, **turn)
    page = rng.choice([1, 8, 16, 20, 32, 64, 100, 128])
    slots_first = rng.random() < 0.5
    b = size(1, 64)
    if op == "append":
        n = rng.choice([1, 1, 3, size(1, 4000)])
        b = max(1, min(b, 16000 // n))
        return _append(b=b, n=n, ragged=rng.random() < 0.5, most=n + size(1, 1000), page=page, slots_first=slots_first,
                       **common, **turn)
    # the keys of the largest listed case at most, by the bytes of one of them
    item = 4 if io == "fp32" else 2
    most = size(1, max(100, min(32768, (8 * 32768 * 8 * 128 * 2) // (2 * b * hk * d * item))))
    n = 1 if op == "step" else rng.choice([1, 1, 1, 4, 7])
    case = _paged(b=b, n=n, ragged=n > 1 and rng.random() < 0.5, most=max(most, n), page=page, slots_first=slots_first,
                  cap=rng.choice([0.0, 0.0, 30.0, 50.0]), radius=rng.choice([0, 0, 32, 128]), **common)
    return {**case, "op": "step", **turn} if op == "step" else case


# ----------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------
def _lengths(case):
    """Keys of each sequence: the most in one, less in the others; and how many of them are new."""
    r = random.Random("lengths %d %d %d" % (case["b"], case["n"], case["most"]))
    n, most = case["n"], case["most"]
    lengths = [most] + [r.randint(max(n, most // 4), most) for _ in range(case["b"] - 1)]
    counts = [n] + [r.randint(0 if n < 8 else n // 8, n) if case["ragged"] else n for _ in range(case["b"] - 1)]
    return lengths, counts


def _frequencies(rot, factor):
    """Radians a position of each pair; for contexts ``factor`` times as long the slow ones are slowed: those that turn
    at most once over 4096 positions by the whole factor, those that turn 32 times not, linearly in between."""
    out = []
    for i in range(rot // 2):
        f = 10000.0 ** (-2.0 * i / rot)
        keep = min(max((4096 * f / (2 * math.pi) - 1.0) / 31.0, 0.0), 1.0)
        out.append(f * (keep + (1.0 - keep) / factor))
    return torch.tensor(out, dtype=F64)


def _bucket_map(radius):
    """Buckets of the offsets -radius .. radius: exact up to a quarter of them, then logarithmic; both directions."""
    if radius <= 32:
        return list(range(2 * radius + 1))
    exact, half = 16, 32
    side = [d if d < exact else min(half - 1, exact + math.floor(math.log(d / exact) / math.log(radius / exact) * (half - exact)))
            for d in range(radius + 1)]
    return [half + b for b in side[:0:-1]] + side


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = F32 if case["io"] == "fp32" else BF16
    b, n, h, hk, d, op = (case[k] for k in ("b", "n", "h", "hk", "d", "op"))

    def rand(*shape):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=F32).to(dt)

    s = {"case": case, "q": rand(b, n, h, d)}
    if op != "attn":
        s["k"] = rand(b, n, hk, d)
        s["frequencies"] = _frequencies(case["rot"], case["factor"]).to(DEVICE)
        s["magnitude"] = 0.1 * math.log(case["factor"]) + 1.0
    if op == "rotary":
        # positions start anew with every packed sequence
        at = torch.arange(n, device=DEVICE, dtype=I32)
        if case["docs"]:
            first = (at * case["docs"]) // n
            at = at - (first * n + case["docs"] - 1) // case["docs"]
        s["positions"] = (at + case["start"]).to(I32).expand(b, n).contiguous()
        if case["train"]:
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
            s["dq"], s["dk"] = rand(b, n, h, d), rand(b, n, hk, d)
        return s
    if op != "attn":
        s["v"] = rand(b, n, hk, d)
    # pages of all sequences in any order, a few of nobody among them; table entries past a sequence's end name none
    lengths, counts = _lengths(case)
    page, most = case["page"], case["most"]
    used = [-(-length // page) for length in lengths]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((b, -(-most // page)), -1, dtype=I32)
    for i, u in enumerate(used):
        table[i, :u] = torch.tensor(order[sum(used[:i]):sum(used[:i + 1])], dtype=I32)
    s["table"] = table.to(DEVICE)
    s["lengths"] = torch.tensor(lengths, dtype=I32, device=DEVICE)
    s["counts"] = torch.tensor(counts, dtype=I32, device=DEVICE) if case["ragged"] else None
    for name in ("keys", "values"):   # [pages, page, Hk, D], in memory with the heads or the slots of a page outside
        s[name] = rand(pages, page, hk, d) if case["slots_first"] else rand(pages, hk, page, d).transpose(1, 2)
    if op != "append":
        s["cap"] = case["cap"] or None
        s["bias"] = s["buckets"] = None
        if case["radius"]:
            buckets = _bucket_map(case["radius"])
            s["buckets"] = torch.tensor(buckets, dtype=torch.uint8, device=DEVICE)
            s["bias"] = (0.5 * torch.randn(max(buckets) + 1, h, generator=g, device=DEVICE)).to(dt)
    return s


# ----------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------
def _angles(s, positions):
    """cos and sin [B, N, 1, rot / 2], rounded to fp32 last."""
    a = positions.double()[:, :, None, None] * s["frequencies"]
    return (a.cos() * s["magnitude"]).float(), (a.sin() * s["magnitude"]).float()


def _turn(x, cos, sin, interleaved, back=False):
    rot = 2 * cos.shape[-1]
    x = x.detach().float()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    if back:
        sin = -sin
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _rotary_plain(s):
    cos, sin = _angles(s, s["positions"])
    il, dt = s["case"]["interleaved"], s["q"].dtype
    out = [_turn(s[n], cos, sin, il).to(dt) for n in ("q", "k")]
    if s["case"]["train"]:
        out += [_turn(s[n], cos, sin, il, True).to(dt) for n in ("dq", "dk")]
    return out


def _new(s):
    """Positions of the new tokens [B, N], and which of them are there."""
    n, dev = s["case"]["n"], s["lengths"].device
    counts = s["counts"] if s["counts"] is not None else torch.full_like(s["lengths"], n)
    i = torch.arange(n, device=dev)
    return (s["lengths"] - counts).long()[:, None] + i, i < counts[:, None]


def _append_plain(s):
    pos, there = _new(s)
    cos, sin = _angles(s, pos)
    il, dt, page = s["case"]["interleaved"], s["q"].dtype, s["case"]["page"]
    q = torch.where(there[:, :, None, None], _turn(s["q"], cos, sin, il), 0.0).to(dt)
    k = _turn(s["k"], cos, sin, il).to(dt)
    row = torch.gather(s["table"].long(), 1, (pos // page).clamp(0, s["table"].shape[1] - 1))[there]
    slot = (pos % page)[there]
    s["keys"][row, slot] = k[there]
    s["values"][row, slot] = s["v"][there]
    return s["keys"], s["values"], q


def _attn_plain(s, q):
    case = s["case"]
    b, n, h, hk, d = (case[k] for k in ("b", "n", "h", "hk", "d"))
    which = s["table"].long().clamp(min=0)
    k, v = (s[name][which].reshape(b, -1, hk, d).transpose(1, 2).float() for name in ("keys", "values"))   # [B, Hk, L, D]
    pos, there = _new(s)
    j = torch.arange(k.shape[2], device=pos.device)
    ok = (j <= pos[:, :, None]) & there[:, :, None]                       # [B, N, L]
    q = q.float().view(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4)       # [B, Hk, G, N, D]
    sc = torch.matmul(q.reshape(b, hk, -1, d), k.transpose(2, 3).contiguous()).view(b, hk, h // hk, n, -1) * d ** -0.5
    if s["cap"]:
        sc = s["cap"] * torch.tanh(sc / s["cap"])
    if s["bias"] is not None:
        radius = case["radius"]
        idx = s["buckets"].long()[(j - pos[:, :, None]).clamp(-radius, radius) + radius]
        sc = sc + s["bias"].float()[idx].view(b, n, -1, hk, h // hk).permute(0, 3, 4, 1, 2)
    ok = ok[:, None, None]
    sc = sc.masked_fill(~ok, -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    v = torch.where(ok.any((1, 2, 3))[:, None, :, None], v, 0.0)
    o = torch.matmul(p.reshape(b, hk, -1, p.shape[-1]), v).view(b, hk, h // hk, n, d)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(s["q"].dtype)


def _run_own(s):
    case, op = s["case"], s["case"]["op"]
    if op == "rotary":
        from bioemu2_amd.rotary import rotary

        def call():
            return rotary(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=case["interleaved"],
                          magnitude=s["magnitude"])

        if not case["train"]:
            with torch.no_grad():
                return call()
        q, k = call()
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    from bioemu2_amd.paged_cache import paged_append, paged_attention

    q = s["q"]
    with torch.no_grad():
        if op != "attn":
            q = paged_append(s["keys"], s["values"], s["k"], s["v"], s["table"], s["lengths"], counts=s["counts"], q=q,
                             frequencies=s["frequencies"], interleaved=case["interleaved"], magnitude=s["magnitude"])
        if op == "append":
            return s["keys"], s["values"], q
        o = paged_attention(q, s["keys"], s["values"], s["table"], s["lengths"], counts=s["counts"], cap=s["cap"],
                            bias_table=s["bias"], bias_buckets=s["buckets"])
    return o if op == "attn" else (s["keys"], s["values"], q, o)


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "rotary":
        return _rotary_plain(state)
    if op == "append":
        return _append_plain(state)
    if op == "attn":
        return _attn_plain(state, state["q"])
    keys, values, q = _append_plain(state)
    return keys, values, q, _attn_plain(state, q)


# ----------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------
def work(case):
    item = 4 if case["io"] == "fp32" else 2
    b, n, h, hk, d, op = (case[k] for k in ("b", "n", "h", "hk", "d", "op"))
    if op == "rotary":
        values = b * n * (h + hk) * (2 if case["train"] else 1)
        return {"bytes": float(2 * values * d * item), "flops": float(3 * values * case["rot"])}
    lengths, counts = _lengths(case)
    new = sum(counts)
    w = {"bytes": 0.0, "flops": 0.0}
    if op != "attn":   # q, k and v in and out
        w["bytes"] += 2 * new * (h + 2 * hk) * d * item
        w["flops"] += 3 * new * (h + hk) * case["rot"]
    if op != "append":
        keys = sum(length for length, c in zip(lengths, counts) if c)
        pairs = sum(c * length - c * (c - 1) // 2 for length, c in zip(lengths, counts))
        w["bytes"] += (2 * keys * hk + 2 * b * n * h) * d * item
        w["flops"] += 4 * pairs * h * d
    return w


# ----------------------------------------------------------------------------
# The same results in float64
# ----------------------------------------------------------------------------
def _rotate64(s, x, positions, sign=1.0):
    """x [B, N, heads, D] as complex numbers times magnitude e^(i position frequency)."""
    rot = s["case"]["rot"]
    x = x.detach().double()
    turn = torch.polar(torch.full((), s["magnitude"], dtype=F64, device=x.device).expand(*positions.shape, rot // 2),
                       sign * positions.double()[..., None] * s["frequencies"])[:, :, None]
    head = x[..., :rot]
    if s["case"]["interleaved"]:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous()) * turn
        head = torch.cat((z.real, z.imag), -1)
    return torch.cat((head, x[..., rot:]), -1)


def _append64(s):
    case = s["case"]
    lengths, counts = _lengths(case)
    keys, values = s["keys"].double(), s["values"].double()
    q = torch.zeros(s["q"].shape, dtype=F64, device=DEVICE)
    table = s["table"].cpu()
    for i, (length, count) in enumerate(zip(lengths, counts)):
        if not count:
            continue
        at = torch.arange(length - count, length)
        where = (table[i][at // case["page"]].long().to(DEVICE), (at % case["page"]).to(DEVICE))
        at = at.to(DEVICE)[None]
        q[i, :count] = _rotate64(s, s["q"][i:i + 1, :count], at)[0]
        keys[where] = _rotate64(s, s["k"][i:i + 1, :count], at)[0]
        values[where] = s["v"][i, :count].double()
    return keys, values, q


def _attn64(s, q, keys, values):
    """``q`` and the caches as the operator reads them."""
    case = s["case"]
    n, h, hk, d, page = (case[k] for k in ("n", "h", "hk", "d", "page"))
    lengths, counts = _lengths(case)
    o = torch.zeros(q.shape, dtype=F64, device=DEVICE)
    for i, (length, count) in enumerate(zip(lengths, counts)):
        if not count:
            continue
        rows = s["table"][i, :-(-length // page)].long()
        k, v = (c[rows].flatten(0, 1)[:length].double() for c in (keys, values))    # [length, Hk, D]
        at = torch.arange(length - count, length, device=DEVICE)[:, None]
        off = torch.arange(length, device=DEVICE)[None] - at                        # [count, length]
        for head in range(h):
            x = q[i, :count, head].double() @ k[:, head * hk // h].T / math.sqrt(d)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if s["bias"] is not None:
                r = case["radius"]
                x = x + s["bias"][:, head].double()[s["buckets"][torch.clamp(off, -r, r) + r].long()]
            o[i, :count, head] = torch.softmax(x.masked_fill(off > 0, -math.inf), -1) @ v[:, head * hk // h]
    return o


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        out = [_rotate64(s, s[n], s["positions"]) for n in ("q", "k")]
        if case["train"]:
            out += [_rotate64(s, s[n], s["positions"], -1.0) for n in ("dq", "dk")]
        return out
    if case["op"] == "attn":
        return _attn64(s, s["q"], s["keys"], s["values"])
    keys, values, q = _append64(s)
    if case["op"] == "append":
        return keys, values, q
    # the step's attention reads what was rounded on the way
    dt = s["q"].dtype
    return keys, values, q, _attn64(s, q.to(dt), keys.to(dt), values.to(dt))
