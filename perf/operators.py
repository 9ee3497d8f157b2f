"""Cases and plain forms of the operators around a key/value cache that is held in 8 bits.

The cache keeps a request's keys and values in pages of ``page`` tokens.  Per page and kv head there is one scale
``s = 2^e``, for keys and for values each; a code ``c`` (0..255) stands for ``(c - 127.5) * s`` and is made by
``floor(x / s) + 128``.  A page's exponent is the largest of its tokens' ``floor(log2(max |x|)) - 6`` (at least -120);
when a later token raises it by d, the codes of the rows before move to ``((c - 128) >> d) + 128``.  A token at the
first row of a page starts the page anew.

Three operators: ``append`` (rotate q and k of a finished product by the tokens' positions, write q out, code k and v
into the pages; read back here with the operator that widens pages, so that the state is seen as the values it stands
for), ``single`` (attention of single tokens, one per request) and ``portion`` (attention of prompt portions whose keys
are in the cache already).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
LOWEST = -120                  # smallest exponent of a scale


# ---- the cases -----------------------------------------------------------------------------------------------

def _case(name, op, lens, starts, nh, nkv, hd, page=16, window=0, cap=50.0, layout="half", rot=0, amplitude=1.0,
          theta=10000.0, scaled=False):
    return {"name": name, "op": op, "lens": lens, "starts": starts, "nh": nh, "nkv": nkv, "hd": hd, "page": page,
            "window": window, "cap": cap, "layout": layout, "rot": rot or hd, "amplitude": amplitude, "theta": theta,
            "scaled": scaled}


def listed():
    return [
        # one request decodes: the append of one token, where latency counts
        _case("append_1_token", "append", "1", "1999", 8, 4, 256),
        # 64 requests decode at contexts of 130 to 8000
        _case("append_64_tokens", "append", "1x64", "130..8000", 16, 8, 256),
        # a prompt portion of 2048 tokens that starts a request
        _case("append_portion", "append", "2048", "0", 8, 4, 256),
        # a mixed step: decoding requests beside portions that begin inside pages; adjacent pairs turned, half of the
        # head, frequencies scaled for long contexts at far positions
        _case("append_mixed_far", "append", "1x5,700,33,1,258", "40000..120000", 32, 16, 128, layout="interleaved",
              rot=64, amplitude=1.2, theta=500000.0, scaled=True),
        # one request decodes at a context of 2000
        _case("single_1x2000", "single", "1", "1999", 8, 4, 256),
        # 64 requests decode at contexts about 2200
        _case("single_64x2200", "single", "1x64", "2100..2300", 16, 8, 256),
        # 56 requests of very different length, keys from a window of 4096
        _case("single_56_uneven", "single", "1x56", "200..4600", 16, 8, 256, window=4096),
        # 16 requests past 4096 with many kv heads of 128
        _case("single_16x4200", "single", "1x16", "4150..4250", 32, 16, 128),
        # a prompt of 4096 tokens in one portion
        _case("portion_4096", "portion", "4096", "0", 16, 8, 256),
        # the last portion of a long prompt: 250 tokens, 7900 in the cache
        _case("portion_250_at_7900", "portion", "250", "7900", 16, 8, 256),
        # portions of several requests with a window, begun inside pages
        _case("portion_ragged", "portion", "5,900,77,1300", "300..3000", 32, 16, 128, window=1024),
        # a few tokens behind a short context
        _case("portion_5_at_300", "portion", "5", "300", 8, 4, 256, cap=0.0),
    ]


HEADS = [(8, 4, 256), (16, 8, 256), (32, 16, 128), (4, 1, 64), (6, 2, 48), (12, 2, 128), (8, 8, 96), (5, 1, 80)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "single", "portion"])
    nh, nkv, hd = rng.choice(HEADS)
    page = rng.choice([16, 16, 32, 64])
    window = rng.choice([0, 0, _log(rng, 100, 4096)])
    cap = rng.choice([0.0, 30.0, 50.0])
    layout = rng.choice(["half", "half", "interleaved"])
    rot = rng.choice([hd, hd, hd // 2])
    extra = dict(page=page, window=window, cap=cap, layout=layout, rot=rot, amplitude=rng.choice([1.0, 1.0, 1.3]),
                 theta=rng.choice([10000.0, 500000.0]), scaled=rng.random() < 0.3)
    if op == "append":
        if rng.random() < 0.5:
            lens, n = "1x%d" % _log(rng, 1, 128), 1
        else:
            lens = ",".join(str(_log(rng, 1, 1200)) for _ in range(rng.randint(1, 3)))
        first = _log(rng, 1, 100000)
        starts = "%d..%d" % (rng.choice([0, first]), first + _log(rng, 1, 8000))
    elif op == "single":
        n = _log(rng, 1, 64)
        lens = "1x%d" % n
        top = _log(rng, 20, min(4600, 140000 // n))
        starts = "%d..%d" % (rng.choice([0, top // 2, int(0.9 * top)]), top)
    else:
        lens = ",".join(str(_log(rng, 2, 900)) for _ in range(rng.randint(1, 3)))
        top = _log(rng, 1, 2500)
        starts = "%d..%d" % (rng.choice([0, top // 2, top]), top)
    c = _case("", op, lens, starts, nh, nkv, hd, **extra)
    del c["name"]
    return c


def _lengths(case):
    """Tokens that every request brings."""
    out = []
    for part in case["lens"].split(","):
        n, _, times = part.partition("x")
        out += [int(n)] * int(times or 1)
    return out


def _starts(case, n):
    """Tokens that every request has in the cache already: spread evenly over the range, in a fixed odd order."""
    lo, _, hi = case["starts"].partition("..")
    lo, hi = int(lo), int(hi or lo)
    if n == 1:
        return [hi]
    vals = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return [vals[(i * 7 + 3) % n] if n % 7 else vals[(i * 11 + 3) % n] for i in range(n)]


def _geometry(case):
    """(lengths, starts, per request the first page and one past the last page that the operator touches)."""
    lens = _lengths(case)
    starts = _starts(case, len(lens))
    P = case["page"]
    reach = 1 if case["op"] == "append" else case["window"]
    spans = []
    for n, s in zip(lens, starts):
        first = max(0, s - reach + 1) if reach else 0
        spans.append((first // P, (s + n - 1) // P + 1))
    return lens, starts, spans


def _keys(case):
    lens, starts, _ = _geometry(case)
    w = case["window"]
    total = 0
    for n, s in zip(lens, starts):
        total += sum(min(p + 1, w) if w else p + 1 for p in range(s, s + n))
    return total


# ---- the inputs ----------------------------------------------------------------------------------------------

def _turns(case):
    """Turns per position of every pair: theta^(-2j/rot) / 2 pi; ``scaled``: the slow pairs' turn eight times slower, the
    fast ones' as they are, a ramp between them (by the wavelength against a context of 8192)."""
    rot = case["rot"]
    f = case["theta"] ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if case["scaled"]:
        wavelength = 2.0 * np.pi / f
        keep = np.clip((8192.0 / wavelength - 1.0) / 3.0, 0.0, 1.0)
        f = f * keep + (1.0 - keep) * f / 8.0
    return f / (2.0 * np.pi)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    nh, nkv, hd, P = case["nh"], case["nkv"], case["hd"], case["page"]
    lens, starts, spans = _geometry(case)
    T, R = sum(lens), len(lens)
    pages = sum(b - a for a, b in spans)
    order = torch.randperm(pages, device="cpu", generator=torch.Generator().manual_seed(int(seed)))
    table = torch.full((R, max(b for _, b in spans)), -1, dtype=torch.int32)
    at = 0
    for r, (a, b) in enumerate(spans):
        table[r, a:b] = order[at:at + b - a].to(torch.int32)
        at += b - a
    cu = np.concatenate([[0], np.cumsum(lens)])
    s = dict(case, tokens=T, requests=R, pages=pages, max_len=max(lens),
             max_context=max(n + p for n, p in zip(lens, starts)),
             contexts=[p + 1 for n, p in zip(lens, starts)] if max(lens) == 1 else [])
    s["positions"] = torch.from_numpy(np.concatenate([np.arange(p, p + n) for n, p in zip(lens, starts)]).astype(np.int32)).to(DEV)
    s["token_seq"] = torch.from_numpy(np.repeat(np.arange(R), lens).astype(np.int32)).to(DEV)
    s["cu_seqlens"] = torch.from_numpy(cu.astype(np.int32)).to(DEV)
    s["seq_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["table"] = table.to(DEV)
    # what the cache holds: keys with some wide channels, values of about unit size, a page apart from its neighbours
    wide = 1.0 + 3.0 * (torch.rand(nkv, 1, hd, device=DEV, generator=g) < 0.05)
    for name, chan in (("k", wide), ("v", torch.ones_like(wide))):
        x = torch.randn(pages, nkv, P, hd, device=DEV, generator=g) * chan
        x *= torch.exp(0.3 * torch.randn(pages, nkv, 1, 1, device=DEV, generator=g))
        e = torch.frexp(x.abs().amax((2, 3)))[1] - 7
        s[name + "_scale"] = torch.ldexp(torch.ones_like(x[:, :, 0, 0]), e)
        s[name] = (torch.floor(torch.ldexp(x, -e[:, :, None, None])) + 128).to(torch.uint8)
        s[name + "_wide"] = torch.zeros(pages, nkv, P, hd, dtype=torch.bfloat16, device=DEV)
        del x
    if case["op"] == "append":
        chan = torch.cat([wide.new_ones(nh, hd), wide[:, 0], wide.new_ones(nkv, hd)])
        s["qkv"] = (torch.randn(T, nh + 2 * nkv, hd, device=DEV, generator=g) * chan).reshape(T, -1)
        s["turns"] = torch.from_numpy(_turns(case)).to(DEV)
    else:
        s["q"] = (1.5 * torch.randn(T, nh * hd, device=DEV, generator=g)).to(torch.bfloat16)
    s["multiplier"] = 1.0 / math.sqrt(hd)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------

def _rotate(x, cos, sin, rot, layout):
    """The first ``rot`` dims of every head turned in pairs."""
    y = x.clone()
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_append(s):
    T, nh, nkv, hd, P = s["tokens"], s["nh"], s["nkv"], s["hd"], s["page"]
    pos = s["positions"].long()
    turn = pos.double()[:, None] * s["turns"][None, :]
    angle = 2.0 * math.pi * (turn - torch.round(turn))
    cos = (s["amplitude"] * torch.cos(angle)).float()[:, None, :]
    sin = (s["amplitude"] * torch.sin(angle)).float()[:, None, :]
    x = s["qkv"].view(T, nh + 2 * nkv, hd)
    qk = _rotate(x[:, :nh + nkv], cos, sin, s["rot"], s["layout"])
    q = qk[:, :nh].reshape(T, nh * hd).to(torch.bfloat16)
    page = s["table"][s["token_seq"].long(), pos // P].long()
    off = pos % P
    first = torch.full((s["pages"],), P, dtype=torch.long, device=DEV).scatter_reduce(0, page, off, "amin")
    rows = torch.arange(P, device=DEV)
    out = []
    for new, codes, scale, to in ((qk[:, nh:], s["k"], s["k_scale"], s["k_wide"]),
                                  (x[:, nh + nkv:], s["v"], s["v_scale"], s["v_wide"])):
        top = torch.zeros(s["pages"], nkv, device=DEV).scatter_reduce(0, page[:, None].expand(T, nkv), new.abs().amax(2), "amax")
        fresh = torch.where(top > 0, torch.frexp(top)[1] - 7, LOWEST).clamp(min=LOWEST)
        before = torch.where((first == 0)[:, None], LOWEST, torch.frexp(scale)[1] - 1)
        e = torch.maximum(before, fresh)
        moved = ((codes.int() - 128) >> (e - before).clamp(max=31)[:, :, None, None].int()) + 128
        earlier = (rows[None, :] < first[:, None])[:, None, :, None]
        codes.copy_(torch.where(earlier, moved, codes.int()))
        codes[page, :, off] = (torch.floor(torch.ldexp(new, -e[page][:, :, None])) + 128).to(torch.uint8)
        scale.copy_(torch.ldexp(torch.ones_like(scale), e))
        to.copy_((codes.float() - 127.5) * scale[:, :, None, None])
        out.append(to)
    return q, out[0], out[1]


def _plain_attention(s):
    """All requests at once, padded to the longest."""
    R, nh, nkv, hd, P = s["requests"], s["nh"], s["nkv"], s["hd"], s["page"]
    G, L, N = nh // nkv, s["max_len"], s["table"].shape[1]
    start, cu = s["seq_start"].long(), s["cu_seqlens"].long()
    place = torch.arange(L, device=DEV)
    row = (cu[:-1, None] + place).clamp(max=s["tokens"] - 1)                          # [R, L]
    there = place[None, :] < (cu[1:] - cu[:-1])[:, None]
    q = s["q"].float().view(-1, nkv, G, hd)[row].permute(0, 2, 3, 1, 4).reshape(R, nkv, G * L, hd)
    held = s["table"].long().clamp(min=0)

    def keys_of(codes, scale):
        x = (codes[held].float() - 127.5) * scale[held][..., None, None]              # [R, N, nkv, P, hd]
        return x.transpose(1, 2).reshape(R, nkv, N * P, hd)

    x = torch.matmul(q, keys_of(s["k"], s["k_scale"]).transpose(2, 3)) * s["multiplier"]
    if s["cap"] > 0:
        x = s["cap"] * torch.tanh(x / s["cap"])
    key = torch.arange(N * P, device=DEV)
    at = (start[:, None] + place)[:, None, :, None]                                   # [R, 1, L, 1]
    seen = (key <= at) & (key > at - s["window"]) if s["window"] else key <= at
    x = x.view(R, nkv, G, L, N * P).masked_fill(~seen[:, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(R, nkv, G * L, N * P), keys_of(s["v"], s["v_scale"]))
    y = y.view(R, nkv, G, L, hd).permute(0, 3, 1, 2, 4).reshape(R, L, nh * hd)
    return y[there].to(torch.bfloat16)


# ---- one pass ------------------------------------------------------------------------------------------------

_kept = {}


def _runtime():
    if "rt" not in _kept:
        from glint_b200.runtime import Runtime
        _kept["rt"] = Runtime(DEV, "bfloat16")
    return _kept["rt"]


def _own(s):
    from glint_b200 import ops_cache8
    rt = _runtime()
    if "handles" not in s:        # what an engine keeps: the layer's cache, and the arrays of a step
        s["handles"] = (ops_cache8.Cache8(s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_wide"], s["v_wide"]),
                        ops_cache8.StepArrays(s["positions"], s["token_seq"], s["seq_start"], s["cu_seqlens"], s["table"],
                                              s["max_len"], s["max_context"], contexts=s["contexts"]))
    cache, step = s["handles"]
    step.begin()                  # a new step: nothing that an earlier one planned is used again
    if s["op"] == "append":
        q = ops_cache8.append(rt, cache, step, s["qkv"], s["turns"], s["nh"], layout=s["layout"], amplitude=s["amplitude"])
        k, v = ops_cache8.unpack(rt, cache, step, window=1)
        return q, k, v
    return ops_cache8.attention(rt, cache, step, s["q"], s["nh"], s["multiplier"], softcap=s["cap"], window=s["window"])


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["op"] == "append" else _plain_attention(state)


def work(case):
    nh, nkv, hd, P = case["nh"], case["nkv"], case["hd"], case["page"]
    lens, _, spans = _geometry(case)
    T, pages = sum(lens), sum(b - a for a, b in spans)
    held = 2 * pages * nkv * (P * hd + 4)                      # codes and scales of the pages
    if case["op"] == "append":
        return {"bytes": 4 * T * (nh + 2 * nkv) * hd + 2 * T * nh * hd + 2 * T * nkv * hd + held + 4 * pages * nkv * P * hd,
                "flops": 3 * T * (nh + nkv) * case["rot"] + 4 * T * nkv * hd}
    return {"bytes": held + 4 * T * nh * hd, "flops": 4 * nh * hd * _keys(case)}


# ---- the definition in 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    lens, starts, _ = _geometry(case)
    nh, nkv, hd, P = case["nh"], case["nkv"], case["hd"], case["page"]
    table = s["table"].cpu().numpy()
    if case["op"] != "append":
        if 4.0 * nh * hd * _keys(case) > 2e12:
            return None
        held = {n: (s[n].double() * 2.0 - 255.0) * (0.5 * s[n + "_scale"].double())[:, :, None, None] for n in ("k", "v")}
        got, t = [], 0
        for r, (n, p) in enumerate(zip(lens, starts)):
            lo = max(0, p - case["window"] + 1) // P if case["window"] else 0
            ids = torch.from_numpy(table[r, lo:(p + n - 1) // P + 1].astype(np.int64)).to(DEV)
            k, v = (held[m][ids].transpose(0, 1).reshape(nkv, -1, hd) for m in ("k", "v"))
            key = lo * P + torch.arange(k.shape[1], device=DEV)
            for a in range(0, n, 256):
                b = min(n, a + 256)
                at = torch.arange(p + a, p + b, device=DEV)[:, None]
                off = (key[None] > at) | ((key[None] <= at - case["window"]) if case["window"] else (key[None] < 0))
                q = s["q"][t + a:t + b].double().view(b - a, nkv, nh // nkv, hd)
                x = torch.einsum("tkgd,kld->kgtl", q, k) / math.sqrt(hd)
                x = case["cap"] * torch.tanh(x / case["cap"]) if case["cap"] else x
                x = x.masked_fill(off, -math.inf)
                got.append(torch.einsum("kgtl,kld->tkgd", torch.softmax(x, -1), v).reshape(b - a, nh * hd))
            t += n
        return torch.cat(got)
    rot, T = case["rot"], sum(lens)
    x = s["qkv"].double().cpu().numpy().reshape(T, nh + 2 * nkv, hd)
    pos = np.concatenate([np.arange(p, p + n) for n, p in zip(lens, starts)])
    z = case["amplitude"] * np.exp(2j * np.pi * np.mod(pos[:, None] * _turns(case)[None], 1.0))[:, None, :]
    ia, ib = (np.arange(rot // 2), np.arange(rot // 2) + rot // 2) if case["layout"] == "half" else \
        (np.arange(0, rot, 2), np.arange(1, rot, 2))
    w = (x[:, :nh + nkv, ia] + 1j * x[:, :nh + nkv, ib]) * z
    x[:, :nh + nkv, ia], x[:, :nh + nkv, ib] = w.real, w.imag
    out = [torch.from_numpy(x[:, :nh].reshape(T, nh * hd).copy())]
    for name, at in (("k", nh), ("v", nh + nkv)):
        c = s[name].cpu().numpy().astype(np.float64) - 128.0
        e = np.frexp(s[name + "_scale"].cpu().numpy())[1] - 1
        t = 0
        for r, (n, p) in enumerate(zip(lens, starts)):
            for lo in range(p - p % P, p + n, P):              # page by page
                a, b = max(lo, p), min(lo + P, p + n)
                y = x[t + a - p:t + b - p, at:at + nkv].transpose(1, 0, 2)
                i = table[r, lo // P]
                big = np.abs(y).max((1, 2))
                need = np.where(big > 0, np.maximum(np.frexp(big)[1] - 7, LOWEST), LOWEST)
                new = need if a == lo else np.maximum(need, e[i])
                c[i, :, :a - lo] = np.floor(c[i, :, :a - lo] / 2.0 ** (new - e[i])[:, None, None]) if a > lo else 0.0
                c[i, :, a - lo:b - lo] = np.floor(y / 2.0 ** new[:, None, None])
                e[i] = new
            t += n
        out.append(torch.from_numpy((c + 0.5) * 2.0 ** e[:, :, None, None].astype(np.float64)))
    return tuple(out)
