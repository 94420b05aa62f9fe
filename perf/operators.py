"""Cases that measure the serving operators: rotary positions (and their gradient), appending new tokens to a paged cache,
attention over that cache, and the handling of its pages.

`run` computes each operator in plain torch operations (32-bit, angles in 64), or, where `own` is set, with the calls a
user makes of `triton_ext_b200.rotary` and `triton_ext_b200.paged`. `exact` is the operator's definition in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
DEV = "cuda"


# ---- cases -----------------------------------------------------------------------------------------------------------
def _rotary(name, z, h, hk, n, d, rd, dtype, interleaved=False, scaling="none", factor=1.0, first=0):
    return dict(name=name, op="rotary", z=z, h=h, hk=hk, n=n, d=d, rd=rd, dtype=dtype, interleaved=interleaved,
                scaling=scaling, factor=factor, first=first)


def _append(name, batch, q_max, kv_max, h, hk, d, rd, page, dtype, interleaved=False, scaling="none", factor=1.0):
    return dict(name=name, op="append", batch=batch, q_max=q_max, kv_max=kv_max, h=h, hk=hk, d=d, rd=rd, page=page,
                dtype=dtype, interleaved=interleaved, scaling=scaling, factor=factor)


def _attend(name, batch, q_max, kv_max, h, hk, d, page, dtype, ragged=True, window=0):
    return dict(name=name, op="attend", batch=batch, q_max=q_max, kv_max=kv_max, h=h, hk=hk, d=d, page=page, dtype=dtype,
                ragged=ragged, window=window)


def listed():
    return [
        # a training step's q and k before attention, forward and backward: the attention benchmark's batch and length
        _rotary("rotary train", 4, 32, 8, 4096, 128, 128, "bf16"),
        # a short odd sequence at far positions of a context stretched by parts, part of the head rotated, pairs interleaved
        _rotary("rotary partial far", 3, 5, 1, 77, 64, 32, "f16", True, "parts", 8.0, 120000),
        # one new token for each of a batch of conversations
        _append("append tokens", 32, 1, 2000, 32, 8, 128, 128, 16, "bf16"),
        # prompts of several requests, of unequal lengths
        _append("append prompts", 6, 2048, 4096, 32, 8, 128, 128, 16, "bf16", False, "linear", 4.0),
        # one conversation, one token: latency is all there is
        _attend("attend one", 1, 1, 777, 16, 4, 64, 16, "f16", False),
        # decoding a batch of conversations of unequal lengths
        _attend("attend batch", 64, 1, 8192, 32, 8, 128, 16, "bf16"),
        # two very long contexts, eight query heads to a key head
        _attend("attend long", 2, 1, 131071, 32, 4, 128, 64, "bf16", False),
        # verifying five drafted tokens a sequence, with a sliding window
        _attend("attend drafts", 16, 5, 4100, 32, 8, 128, 32, "f16", True, 1024),
        # a chunk of a long prompt over what is cached already
        _attend("attend chunk", 1, 2048, 32768, 32, 8, 128, 64, "bf16", False),
        # first chunks of requests of unequal lengths, every head with its own keys
        _attend("attend prompts", 12, 1500, 1700, 12, 12, 64, 16, "f16"),
        # several samples drawn from one prompt: share its pages, copy the last one, make room for the next tokens
        dict(name="pages fork", op="fork", parents=8, children=7, tokens=2000, grow=3, layers=16, hk=8, d=128, page=16, dtype="bf16"),
        # requests end, the rest move together, new ones are admitted
        dict(name="pages compact", op="compact", rows=48, tokens=1000, layers=8, hk=8, d=64, page=32, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "attend", "pages"])
    dtype = rng.choice(["f16", "bf16"])
    d = rng.choice([64, 128])
    hk = rng.choice([1, 2, 4, 5, 8])
    g = rng.choice([1, 2, 3, 4, 6, 8])
    page = rng.choice([16, 32, 64, 128])
    rope = dict(rd=rng.choice([d, d, d // 2, d // 4, 20]), interleaved=rng.random() < 0.5,
                scaling=rng.choice(["none", "linear", "base", "parts"]), factor=rng.choice([2.0, 4.0, 8.0]))
    if rope["scaling"] == "none":
        rope["factor"] = 1.0
    if op == "rotary":
        c = _rotary("", _log(rng, 1, 4), hk * min(g, 4), hk, _log(rng, 1, 2900), d, dtype=rng.choice([dtype, dtype, "f32"]),
                    first=rng.choice([0, 5, 100000, 2000000]), **rope)
    elif op == "append":
        q_max = rng.choice([1, 1, _log(rng, 2, 1500)])
        c = _append("", _log(rng, 1, 64 if q_max == 1 else 6), q_max, q_max + _log(rng, 1, 2000), hk * g, hk, d, page=page,
                    dtype=dtype, **rope)
    elif op == "attend":
        q_max = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 1500)])
        kv_max = q_max + _log(rng, 1, 16000 if q_max <= 16 else 8000)
        batch = _log(rng, 1, 64)
        while batch > 1 and batch * q_max * hk * g * kv_max > 1.2e9 or batch * hk * kv_max * d > 6e8:
            batch -= 1
        c = _attend("", batch, q_max, kv_max, hk * g, hk, d, page, dtype, rng.random() < 0.7,
                    rng.choice([0, 0, 0, _log(rng, 1, 2000)]))
    elif rng.random() < 0.5:
        c = dict(op="fork", parents=_log(rng, 1, 8), children=_log(rng, 1, 7), tokens=_log(rng, 1, 2000), grow=_log(rng, 1, 40),
                 layers=_log(rng, 1, 12), hk=min(hk, 8), d=d, page=page, dtype=dtype)
    else:
        c = dict(op="compact", rows=2 * _log(rng, 1, 20), tokens=_log(rng, 1, 1000), layers=_log(rng, 1, 6), hk=min(hk, 8),
                 d=64, page=page, dtype=dtype)
    c.pop("name", None)
    return c


# ---- what a case fixes besides its contents: lengths and angles ---------------------------------------------------------
def _lengths(c):
    """(new tokens, cached tokens with the new ones) of each sequence; ragged ones lie between a tenth of the largest and it."""
    r = random.Random(1000 * c["batch"] + c["q_max"])
    if not c.get("ragged", True):
        return [c["q_max"]] * c["batch"], [c["kv_max"]] * c["batch"]
    q = [c["q_max"] if c["q_max"] <= 16 else max(1, int(c["q_max"] * r.uniform(0.1, 1.0))) for _ in range(c["batch"])]
    kv = [max(n, int(c["kv_max"] * r.uniform(0.1, 1.0))) for n in q]
    q[0], kv[0] = c["q_max"], c["kv_max"]
    return q, kv


def _row_tokens(c, count):
    r = random.Random(7 * count + c["tokens"])
    return [c["tokens"]] + [max(1, int(c["tokens"] * r.uniform(0.1, 1.0))) for _ in range(count - 1)]


BASE, ORIGINAL, LOW, HIGH = 10000.0, 4096, 1.0, 32.0


def _frequencies(c):
    """(radians per position of each pair, the magnitude of the rotated vector)."""
    rd, s, f = c["rd"], c["scaling"], c["factor"]
    base = BASE * f ** (rd / (rd - 2)) if s == "base" else BASE
    freq = [base ** (-2.0 * i / rd) for i in range(rd // 2)]
    if s == "linear":
        freq = [w / f for w in freq]
    if s == "parts":
        ramp = [min(1.0, max(0.0, (ORIGINAL * w / (2 * math.pi) - LOW) / (HIGH - LOW))) for w in freq]
        freq = [w * (g + (1.0 - g) / f) for w, g in zip(freq, ramp)]
    return freq, (0.1 * math.log(f) + 1.0 if s == "parts" else 1.0)


def _handle(c):
    """The rotary description that a user's program keeps."""
    from triton_ext_b200 import rotary
    more = dict(original_len=ORIGINAL, low=LOW, high=HIGH) if c["scaling"] == "parts" else {}
    return rotary.Rope(c["rd"], base=BASE, interleaved=c["interleaved"], scaling=None if c["scaling"] == "none" else c["scaling"],
                       factor=c["factor"], **more)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32 if dt == torch.float32 else dt)

    def i32(values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    s = {"case": c}
    if "rd" in c:
        freq, s["magnitude"] = _frequencies(c)
        s["freq"] = torch.tensor(freq, dtype=torch.float64, device=DEV)
        s["rope"] = _handle(c) if own else None
    if c["op"] == "rotary":
        # q and k as projections leave them: [batch, tokens, heads, head_dim] in memory, seen as [batch, heads, tokens, head_dim]
        s["q"], s["gq"] = (normal(c["z"], c["n"], c["h"], c["d"]).transpose(1, 2) for _ in range(2))
        s["k"], s["gk"] = (normal(c["z"], c["n"], c["hk"], c["d"]).transpose(1, 2) for _ in range(2))
        s["positions"] = torch.arange(c["first"], c["first"] + c["n"], device=DEV)
        return s
    if c["op"] in ("append", "attend"):
        q_len, kv_len = _lengths(c)
        width = -(-max(kv_len) // c["page"])
        used = [-(-n // c["page"]) for n in kv_len]
        pages = sum(used) + 3
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        col = torch.arange(width, device=DEV)
        first = torch.tensor([0] + used, device=DEV).cumsum(0)[:-1]
        at = first[:, None] + col
        s["table"] = torch.where(col < i32(used)[:, None], order[at.clamp(max=pages - 1)], i32(-1))
        s["kv_lens"] = i32(kv_len)
        s["cu_q"] = torch.tensor([0] + q_len, device=DEV).cumsum(0).to(torch.int32) if c["q_max"] > 1 else None
        s["max_q"], total = c["q_max"], sum(q_len)
        s["k_pages"], s["v_pages"] = (normal(pages, c["page"], c["hk"], c["d"]) for _ in range(2))
        if c["op"] == "append":  # q, k and v are parts of one projection's output
            qkv = normal(total, c["h"] + 2 * c["hk"], c["d"])
            s["q"], s["k"], s["v"] = qkv.split([c["h"], c["hk"], c["hk"]], dim=1)
        else:
            s["q"], s["scale"] = normal(total, c["h"], c["d"]), c["d"] ** -0.5
        return s
    # pages: rows of the table with their tokens, packed from the lowest page on
    rows = c["parents"] * (1 + c["children"]) if c["op"] == "fork" else c["rows"]
    filled = c["parents"] if c["op"] == "fork" else rows
    tokens = _row_tokens(c, filled)
    used = [-(-n // c["page"]) for n in tokens]
    spare = rows * (-(-c["grow"] // c["page"]) + 1) if c["op"] == "fork" else 5
    pages, width = sum(used) + spare, max(used) + (-(-c.get("grow", 0) // c["page"]) + 1)
    s["k"], s["v"] = (normal(c["layers"], pages, c["page"], c["hk"], c["d"]) for _ in range(2))
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    s["table"], s["lens"] = table.to(DEV), i32(tokens + [0] * (rows - filled))
    s["refs"] = i32([1] * sum(used) + [0] * spare)
    if c["op"] == "fork":
        s["children"] = torch.arange(filled, rows, dtype=torch.int32, device=DEV)
        s["sources"] = torch.arange(filled, dtype=torch.int32, device=DEV).repeat_interleave(c["children"])
        s["all"] = torch.arange(rows, dtype=torch.int32, device=DEV)
        s["counts"] = torch.where(s["all"] >= filled, c["grow"], 0).to(torch.int32)
    else:
        half = rows // 2
        s["halves"] = [(torch.arange(a, a + half, dtype=torch.int32, device=DEV), i32(tokens[a:a + half])) for a in (0, half)]
    if own:
        from triton_ext_b200 import paged
        s["cache"] = paged.PagedCache(s["k"], s["v"], s["table"], s["lens"], s["refs"])
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------
def _rotate(x, angle, magnitude, interleaved, rd):
    """x [..., tokens, heads, d] turned by angle [..., tokens, rd / 2]; returns x's type."""
    c, s = (angle.cos() * magnitude).float()[..., None, :], (angle.sin() * magnitude).float()[..., None, :]
    part, rest = x[..., :rd].float(), x[..., rd:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        a, b = part[..., : rd // 2], part[..., rd // 2:]
        turned = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    return torch.cat((turned.to(x.dtype), rest), dim=-1)


def _plain_rotary(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["freq"]

    def turn(x, sign):
        return _rotate(x.transpose(1, 2), angle * sign, s["magnitude"], c["interleaved"], c["rd"]).transpose(1, 2)

    return [turn(s["q"], 1), turn(s["k"], 1), turn(s["gq"], -1), turn(s["gk"], -1)]


def _places(s):
    """(sequence, position in it) of each new token."""
    kv = s["kv_lens"].long()
    if s["cu_q"] is None:
        row = torch.arange(kv.numel(), device=kv.device)
        return row, kv - 1
    cu = s["cu_q"].long()
    token = torch.arange(s["q"].shape[0], device=kv.device)
    row = (token[:, None] >= cu[1:]).sum(1)
    return row, kv[row] - (cu[row + 1] - cu[row]) + (token - cu[row])


def _plain_append(s):
    c = s["case"]
    row, pos = _places(s)
    angle = pos.double()[:, None] * s["freq"]
    q = _rotate(s["q"], angle, s["magnitude"], c["interleaved"], c["rd"])
    k = _rotate(s["k"], angle, s["magnitude"], c["interleaved"], c["rd"])
    page, at = s["table"][row, pos // c["page"]].long(), pos % c["page"]
    s["k_pages"][page, at] = k
    s["v_pages"][page, at] = s["v"]
    return [q, s["k_pages"], s["v_pages"]]


def _plain_attend(s):
    c = s["case"]
    table, kv, q = s["table"].long().clamp(min=0), s["kv_lens"].long(), s["q"]
    batch, most, total = table.shape[0], s["max_q"], q.shape[0]
    k, v = (x[table].flatten(1, 2).float().transpose(1, 2) for x in (s["k_pages"], s["v_pages"]))  # [batch, hk, keys, d]
    j = torch.arange(most, device=q.device)
    cu = s["cu_q"].long() if s["cu_q"] is not None else torch.arange(batch + 1, device=q.device)
    count = cu[1:] - cu[:-1]
    token = torch.where(j < count[:, None], cu[:-1, None] + j, total)  # [batch, most]; the last row of `padded` is for none
    padded = torch.cat((q, q.new_zeros(1, *q.shape[1:])))
    grouped = padded[token].float().view(batch, most, c["hk"], -1, c["d"]).permute(0, 2, 3, 1, 4)  # [batch, hk, group, most, d]
    group = grouped.shape[2]
    scores = grouped.reshape(batch, c["hk"], group * most, c["d"]) @ k.transpose(2, 3)
    scores = scores.mul_(s["scale"]).view(batch, c["hk"], group, most, -1)
    pos = kv[:, None] - count[:, None] + j
    key = torch.arange(k.shape[2], device=q.device)
    seen = key <= pos[..., None]
    if c["window"]:
        seen = seen & (key > pos[..., None] - c["window"])
    seen = (seen & (j < count[:, None])[..., None])[:, None, None]
    top = scores.masked_fill_(~seen, -math.inf).amax(-1, keepdim=True)
    weight = scores.sub_(top.clamp(min=-1e30)).exp_()
    norm = weight.sum(-1, keepdim=True)
    out = (weight.view(batch, c["hk"], group * most, -1) @ v).view(batch, c["hk"], group, most, c["d"])
    out = torch.where(norm > 0, out / norm, 0.0).permute(0, 3, 1, 2, 4).reshape(batch * most, -1, c["d"])
    result = q.new_zeros(total + 1, *q.shape[1:])
    result[token.flatten()] = out.to(q.dtype)
    return result[:total]


def _plain_free(s, rows):
    pages = s["table"][rows.long()].flatten().long()
    s["refs"].index_put_((pages.clamp(min=0),), -(pages >= 0).to(torch.int32), accumulate=True)
    s["table"][rows.long()] = -1
    s["lens"][rows.long()] = 0


def _plain_fork(s, dst, src):
    row, n = s["table"][src.long()], s["lens"][src.long()]
    pages = row.flatten().long()
    _plain_free(s, dst)
    s["refs"].index_put_((pages.clamp(min=0),), (pages >= 0).to(torch.int32), accumulate=True)
    s["table"][dst.long()] = row
    s["lens"][dst.long()] = n


def _plain_reserve(s, rows, counts):
    """Pages for `counts` new tokens in each row, the lowest free ones first; a last page that is shared is copied first, by all
    of its rows but the last that would keep it to itself."""
    page, table, refs = s["case"]["page"], s["table"], s["refs"]
    rows, counts = rows.long(), counts.long()
    n = s["lens"][rows].long()
    have, want = -(-n // page), -(-(n + counts) // page)
    last = table[rows, (have - 1).clamp(min=0)].long()
    part = (n % page > 0) & (counts > 0)
    earlier = ((last[:, None] == last) & part & (torch.arange(len(rows), device=n.device) < torch.arange(len(rows), device=n.device)[:, None])).sum(1)
    copy = part & (refs[last.clamp(min=0)] - earlier > 1)
    need = want - have + copy
    end = need.cumsum(0)
    free = torch.argsort((refs > 0).to(torch.int8), stable=True)
    who = copy.nonzero().flatten()
    src, dst = last[who], free[end[who] - need[who]]
    s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
    refs.index_put_((src,), refs.new_tensor(-1).expand(len(src)), accumulate=True)
    table[rows[who], have[who] - 1] = dst.to(torch.int32)
    col = torch.arange(table.shape[1], device=n.device)
    fresh = (col >= have[:, None]) & (col < want[:, None])
    at = (end - need + copy)[:, None] + col - have[:, None]
    table[rows] = torch.where(fresh, free[at.clamp(0, len(free) - 1)].to(torch.int32), table[rows])
    refs[free] = torch.where(torch.arange(len(free), device=n.device) < end[-1], 1, refs[free])
    s["lens"][rows] = (n + counts).to(torch.int32)


def _plain_compact(s):
    """The live pages at or past the number of live pages go to the holes below it, in order."""
    live = s["refs"] > 0
    index = torch.arange(len(live), device=live.device)
    low = index < live.sum()
    src, dst = (live & ~low).nonzero().flatten(), (~live & low).nonzero().flatten()
    s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
    to = index.to(torch.int32)
    to[src] = dst.to(torch.int32)
    s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].long().clamp(min=0)], -1))
    s["refs"][dst], s["refs"][src] = s["refs"][src], 0


def _plain_pages(s):
    if s["case"]["op"] == "fork":
        _plain_free(s, s["children"])
        _plain_fork(s, s["children"], s["sources"])
        _plain_reserve(s, s["all"], s["counts"])
    else:
        (a, na), (b, nb) = s["halves"]
        _plain_free(s, a)
        _plain_compact(s)
        _plain_reserve(s, a, na)
        _plain_free(s, b)
        _plain_compact(s)
        _plain_reserve(s, b, nb)
    return _state(s)


def _state(s):
    return [s["table"], s["lens"], s["refs"], s["k"], s["v"]]


# ---- the framework's calls -----------------------------------------------------------------------------------------------
def _own(s):
    c = s["case"]
    if c["op"] == "rotary":
        from triton_ext_b200 import rotary
        q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
        q2, k2 = rotary.rotary(q, k, s["positions"], s["rope"])
        gq, gk = torch.autograd.grad((q2, k2), (q, k), (s["gq"], s["gk"]))
        return [q2.detach(), k2.detach(), gq, gk]
    from triton_ext_b200 import paged
    if c["op"] == "append":
        q = paged.append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], rope=s["rope"],
                         cu_q=s["cu_q"])
        return [q, s["k_pages"], s["v_pages"]]
    if c["op"] == "attend":
        return paged.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], s["scale"],
                                     cu_q=s["cu_q"], max_q=s["max_q"], window=c["window"])
    cache = s["cache"]
    if c["op"] == "fork":
        cache.free(s["children"])
        cache.fork(s["children"], s["sources"])
        cache.reserve(s["all"], s["counts"])
    else:
        (a, na), (b, nb) = s["halves"]
        cache.free(a)
        cache.compact()
        cache.reserve(a, na)
        cache.free(b)
        cache.compact()
        cache.reserve(b, nb)
    return _state(s)


def run(s):
    if own:
        return _own(s)
    op = s["case"]["op"]
    return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "fork": _plain_pages,
            "compact": _plain_pages}[op](s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def _visible(q, kv, window):
    """Number of (new token, key) pairs that are not masked."""
    total = 0
    for n, m in zip(q, kv):
        first, last = m - n + 1, m  # keys seen by the first and the last new token, without a window
        if not window or window >= last:
            total += (first + last) * n // 2
        elif window <= first:
            total += window * n
        else:
            total += (first + window - 1) * (window - first) // 2 + window * (last - window + 1)
    return total


def work(c):
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "rotary":
        values = c["z"] * c["n"] * (c["h"] + c["hk"]) * c["d"]
        return {"bytes": 4 * values * size + 8 * c["n"], "flops": 2 * 3 * c["z"] * c["n"] * (c["h"] + c["hk"]) * c["rd"]}
    if c["op"] == "append":
        q, kv = _lengths(c)
        values = sum(q) * (c["h"] + 2 * c["hk"]) * c["d"]
        return {"bytes": 2 * values * size + 4 * (sum(q) + 2 * len(q)), "flops": 3 * sum(q) * (c["h"] + c["hk"]) * c["rd"]}
    if c["op"] == "attend":
        q, kv = _lengths(c)
        read = [min(m, n + c["window"] - 1) if c["window"] else m for n, m in zip(q, kv)]
        bytes_ = 2 * sum(q) * c["h"] * c["d"] * size + 2 * sum(read) * c["hk"] * c["d"] * size + 4 * sum(-(-m // c["page"]) for m in read)
        return {"bytes": bytes_ + 8 * len(q), "flops": 4 * _visible(q, kv, c["window"]) * c["h"] * c["d"]}
    page = 2 * c["layers"] * c["page"] * c["hk"] * c["d"] * size
    if c["op"] == "fork":
        tokens = _row_tokens(c, c["parents"])
        moved = sum(c["children"] for n in tokens if n % c["page"])
        cells = sum(c["children"] * (-(-(n + c["grow"]) // c["page"])) for n in tokens)
        return {"bytes": 2 * moved * page + 4 * 4 * cells, "flops": 0}
    tokens = _row_tokens(c, c["rows"])
    used = [-(-n // c["page"]) for n in tokens]
    a, b = sum(used[: c["rows"] // 2]), sum(used[c["rows"] // 2:])
    return {"bytes": 2 * 2 * min(a, b) * page + 4 * 4 * (a + b), "flops": 0}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------
def _turned(x, pos, s, inverse=False):
    """x [tokens, heads, d] as complex numbers times exp(i p f)."""
    c = s["case"]
    freq, magnitude = _frequencies(c)
    rd, x = c["rd"], x.double().clone()
    phase = pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    unit = torch.polar(torch.full_like(phase, magnitude), -phase if inverse else phase)[:, None]
    pairs = (slice(0, rd, 2), slice(1, rd, 2)) if c["interleaved"] else (slice(0, rd // 2), slice(rd // 2, rd))
    z = torch.complex(x[..., pairs[0]], x[..., pairs[1]]) * unit
    x[..., pairs[0]], x[..., pairs[1]] = z.real, z.imag
    return x


def exact(c, seed):
    if c["op"] in ("fork", "compact"):
        return None  # values are moved, none is computed
    s = prepare(c, seed)
    if c["op"] == "rotary":
        whole = lambda x, inv: torch.stack([_turned(y.transpose(0, 1), s["positions"], s, inv).transpose(0, 1) for y in x])  # noqa: E731
        return [whole(s["q"], False), whole(s["k"], False), whole(s["gq"], True), whole(s["gk"], True)]
    q_len, kv_len = _lengths(c)
    if c["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        turned, at = [], 0
        for i, (n, m) in enumerate(zip(q_len, kv_len)):
            pos = torch.arange(m - n, m, device=DEV)
            page, slot = s["table"][i].long()[pos // c["page"]], pos % c["page"]
            turned.append(_turned(s["q"][at:at + n], pos, s))
            kp[page, slot] = _turned(s["k"][at:at + n], pos, s)
            vp[page, slot] = s["v"][at:at + n].double()
            at += n
        return [torch.cat(turned), kp, vp]
    out, at = torch.zeros_like(s["q"], dtype=torch.float64), 0
    group = c["h"] // c["hk"]
    for i, (n, m) in enumerate(zip(q_len, kv_len)):
        pages = s["table"][i, : -(-m // c["page"])].long()
        k, v = (x[pages].flatten(0, 1)[:m].double() for x in (s["k_pages"], s["v_pages"]))
        key, pos = torch.arange(m, device=DEV), torch.arange(m - n, m, device=DEV)[:, None]
        hidden = (key > pos) | (key <= pos - c["window"] if c["window"] else key > pos)
        for h in range(c["h"]):
            logits = s["q"][at:at + n, h].double() @ k[:, h // group].T * c["d"] ** -0.5
            out[at:at + n, h] = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=-1) @ v[:, h // group]
        at += n
    return out
