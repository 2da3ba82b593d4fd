"""The token-mixing operators of a hybrid decoder step, as measured cases.

Three operators and their forms:

  mrope      rotary positions with several axes on q and k, with k and v
             written into a paged cache (mrope_append_kv)
  attention  one new token per sequence over a paged key-value cache
             (paged_attention_decode)
  delta      the gated delta rule: one token per sequence (gated_delta_step)
             and packed prompts (gated_delta_prefill)

With `own` false `run` computes them in elementary torch operations in fp32,
with `own` true through the package's entry points.  `exact` is the
definition in fp64, written apart from the plain forms.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minicpm-v-4.6-orangepi_b200")


def _lib():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import mcv_b200
    return mcv_b200


# ---- cases ------------------------------------------------------------------

# The full-attention layers of the decoder: 8 query heads (or 16) over 2
# key-value heads of 256, 64 rotated dimensions; the linear layers: 16 heads
# with 128 x 128 states.
_THETA = 1.0e7


def listed():
    return [
        # one text token of one conversation: a call's latency
        {"name": "mrope_decode_1", "op": "mrope", "tokens": 1, "decode": True, "q_heads": 8, "kv_heads": 2, "dim": 256,
         "rotary": 64, "interleaved": True, "page": 16, "gated": True, "idle": 0},
        # a served batch's step, some rows idle
        {"name": "mrope_decode_200", "op": "mrope", "tokens": 200, "decode": True, "q_heads": 16, "kv_heads": 2,
         "dim": 256, "rotary": 64, "interleaved": True, "page": 64, "gated": False, "idle": 9},
        # a long prompt with images
        {"name": "mrope_prompt_8191", "op": "mrope", "tokens": 8191, "decode": False, "q_heads": 8, "kv_heads": 2,
         "dim": 256, "rotary": 64, "interleaved": True, "page": 16, "gated": True, "idle": 0},
        # one conversation, early on
        {"name": "attention_b1_611", "op": "attention", "batch": 1, "longest": 611, "ragged": False, "q_heads": 8,
         "kv_heads": 2, "dim": 256, "page": 16},
        # one conversation over a very long context
        {"name": "attention_b1_131071", "op": "attention", "batch": 1, "longest": 131071, "ragged": False,
         "q_heads": 16, "kv_heads": 2, "dim": 256, "page": 64},
        # a served batch of mixed lengths, empty rows among them; head size 128
        {"name": "attention_b48_ragged", "op": "attention", "batch": 48, "longest": 5003, "ragged": True,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16},
        # a full server: the largest read of the cache
        {"name": "attention_b64_16384", "op": "attention", "batch": 64, "longest": 16384, "ragged": True,
         "q_heads": 8, "kv_heads": 2, "dim": 256, "page": 32},
        # one conversation's token in a linear layer
        {"name": "delta_step_b1", "op": "delta_step", "batch": 1, "slots": 4, "k_heads": 16, "v_heads": 16, "dk": 128,
         "dv": 128, "idle": 0},
        # a served batch's step, some rows idle, shared key heads
        {"name": "delta_step_b160", "op": "delta_step", "batch": 160, "slots": 192, "k_heads": 16, "v_heads": 32,
         "dk": 128, "dv": 128, "idle": 5},
        # a short question
        {"name": "delta_prefill_61", "op": "delta_prefill", "batch": 1, "longest": 61, "ragged": False, "start": False,
         "k_heads": 16, "v_heads": 16, "dk": 128, "dv": 128},
        # one long prompt with images
        {"name": "delta_prefill_8000", "op": "delta_prefill", "batch": 1, "longest": 8000, "ragged": False,
         "start": False, "k_heads": 16, "v_heads": 16, "dk": 128, "dv": 128},
        # packed prompts of several conversations that go on from their states
        {"name": "delta_prefill_packed", "op": "delta_prefill", "batch": 11, "longest": 4099, "ragged": True,
         "start": True, "k_heads": 16, "v_heads": 16, "dk": 128, "dv": 128},
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mrope", "attention", "delta_step", "delta_prefill"])
    if op == "mrope":
        decode = rng.random() < 0.5
        dim = rng.choice([64, 128, 256])
        kv = rng.choice([1, 2, 4])
        return {"op": op, "tokens": _logint(rng, 1, 256 if decode else 8000), "decode": decode,
                "q_heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": dim,
                "rotary": rng.choice([r for r in (32, 64, 128, 256) if r <= dim]),
                "interleaved": rng.random() < 0.5, "page": rng.choice([16, 24, 32, 64]),
                "gated": rng.random() < 0.5, "idle": rng.choice([0, 0, 1, 7]) if decode else 0}
    if op == "attention":
        dim = rng.choice([64, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 5, 8, 16])
        batch = _logint(rng, 1, 128)
        longest = min(_logint(rng, 1, 120000), 16384 * 40 * 512 // (batch * kv * dim))
        return {"op": op, "batch": batch, "longest": max(1, longest), "ragged": batch > 1 and rng.random() < 0.8,
                "q_heads": kv * group, "kv_heads": kv, "dim": dim, "page": rng.choice([16, 24, 32, 64])}
    kh = rng.choice([4, 8, 16])
    vh = kh * rng.choice([1, 2])
    dk, dv = rng.choice([64, 128]), rng.choice([64, 128])
    if op == "delta_step":
        batch = _logint(rng, 1, 160)
        return {"op": op, "batch": batch, "slots": batch + rng.randint(0, 32), "k_heads": kh, "v_heads": vh, "dk": dk,
                "dv": dv, "idle": rng.choice([0, 0, 1, 5])}
    batch = _logint(rng, 1, 16)
    longest = min(_logint(rng, 1, 8000), 32000 // batch, 256000 // (batch * vh))
    return {"op": op, "batch": batch, "longest": max(1, longest), "ragged": batch > 1, "start": rng.random() < 0.5,
            "k_heads": kh, "v_heads": vh, "dk": dk, "dv": dv}


def _sections(case):
    """Frequencies per axis (time, height, width)."""
    half = case["rotary"] // 2
    h = half // 3
    return [half - 2 * h, h, h]


def _lengths(case):
    """Sequence lengths of a case: the longest once, the others spread below
    it, one sequence empty where there are enough of them."""
    n, longest = case["batch"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    out = []
    for i in range(n):
        f = ((i * 7919 + 13) % 997) / 996.0
        out.append(max(1, int(longest * (0.25 + 0.75 * f))))
    out[0] = longest
    if n > 4:
        out[n // 2] = 0 if case["op"] == "attention" else 1
    return out


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7 + 11)
    return g


def _randn(g, *shape, dtype=torch.float16, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _image_positions(tokens):
    """Positions on three axes of a prompt of text and images: text advances
    all axes together; an image of h x w patches keeps the time and walks the
    height and width, and the text after it goes on from the largest."""
    t = torch.zeros(3, tokens, dtype=torch.int64)
    at, pos, side = 0, 0, 7
    while at < tokens:
        n = min(37 + at % 11, tokens - at)
        t[:, at:at + n] = torch.arange(pos, pos + n)
        at, pos = at + n, pos + n
        h, w = side, side + 5
        n = min(h * w, tokens - at)
        if n > 0:
            p = torch.arange(n)
            t[0, at:at + n] = pos
            t[1, at:at + n] = pos + p // w
            t[2, at:at + n] = pos + p % w
            at, pos = at + n, pos + max(h, w)
        side = 7 + (side * 3) % 23
    return t


def _prepare_mrope(case, g, seed):
    n, hq, hk, d, page = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    if case["gated"]:     # the q projection also carries the output gate: [q, gate] per head
        q = _randn(g, n, hq, 2 * d)[:, :, :d]
    else:
        q = _randn(g, n, hq, d)
    kv = _randn(g, n, 2, hk, d)
    k, v = kv[:, 0], kv[:, 1]
    if case["decode"]:
        width = 4
        index = torch.randint(0, width * page, (n,), generator=g, device="cuda", dtype=torch.int32)
        if case["idle"]:
            index[n - min(case["idle"], n - 1):] = -1
        base = torch.randint(0, 262144, (n,), generator=g, device="cuda", dtype=torch.int32)
        positions = torch.stack([base, base, base])
        seq = None
        pages = n * width + 3
        table = torch.randperm(pages, generator=g, device="cuda")[:n * width].reshape(n, width).to(torch.int32)
    else:
        width = (n + page - 1) // page
        index = torch.arange(n, device="cuda", dtype=torch.int32)
        positions = (_image_positions(n) + seed % 97).to(device="cuda", dtype=torch.int32)
        seq = torch.zeros(n, device="cuda", dtype=torch.int32)
        pages = width + 3
        table = torch.randperm(pages, generator=g, device="cuda")[:width].reshape(1, width).to(torch.int32)
    ck = _randn(g, pages, hk, page, d)
    cv = _randn(g, pages, hk, page, d)
    st = {"case": case, "q": q, "k": k, "v": v, "positions": positions.contiguous(), "index": index, "seq": seq,
          "table": table.contiguous(), "ck": ck, "cv": cv,
          "q_out": torch.empty(n, hq, d, dtype=torch.float16, device="cuda")}
    if own:
        m = _lib()
        st["cache"] = m.PagedKVCache(ck, cv)
        st["rope"] = m.MRope(rotary_dim=case["rotary"], sections=_sections(case), interleaved=case["interleaved"],
                             theta=_THETA)
    return st


def _prepare_attention(case, g, seed):
    b, hq, hk, d, page = case["batch"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case)
    need = [(x + page - 1) // page for x in lens]
    width, pages = max(1, max(need)), sum(need) + 5
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, x in enumerate(need):
        table[i, :x] = perm[at:at + x]
        at += x
    st = {"case": case, "q": _randn(g, b, hq, d, scale=2.0), "ck": _randn(g, pages, hk, page, d),
          "cv": _randn(g, pages, hk, page, d), "table": table,
          "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda"),
          "out": torch.empty(b, hq, d, dtype=torch.float16, device="cuda"),
          "lse": torch.empty(b, hq, dtype=torch.float32, device="cuda")}
    if own:
        m = _lib()
        st["cache"] = m.PagedKVCache(st["ck"], st["cv"])
        st["workspace"] = m.paged_attention_workspace(b, hq, hk, d)
    return st


def _gates(g, n, heads):
    """Decays and write strengths as the layer makes them: g = -A softplus(a),
    beta = sigmoid(b)."""
    a = torch.rand(heads, generator=g, device="cuda") * 15 + 1
    dt = torch.exp(torch.rand(heads, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
    jitter = torch.exp(0.5 * torch.randn(n, heads, generator=g, device="cuda"))
    return -(a * dt) * jitter, torch.sigmoid(torch.randn(n, heads, generator=g, device="cuda"))


def _prepare_delta(case, g, seed):
    b, hk, hv, dk, dv = case["batch"], case["k_heads"], case["v_heads"], case["dk"], case["dv"]
    step = case["op"] == "delta_step"
    lens = [1] * b if step else _lengths(case)
    n = sum(lens)
    # q, k and v lie side by side in one row, as the layer's projection leaves them
    row = _randn(g, n, 2 * hk * dk + hv * dv)
    q = row[:, :hk * dk].unflatten(1, (hk, dk))
    k = row[:, hk * dk:2 * hk * dk].unflatten(1, (hk, dk))
    v = row[:, 2 * hk * dk:].unflatten(1, (hv, dv))
    decay, beta = _gates(g, n, hv)
    st = {"case": case, "q": q, "k": k, "v": v, "g": decay, "beta": beta,
          "out": torch.empty(n, hv, dv, dtype=torch.float16, device="cuda")}
    if step:
        slots = case["slots"]
        st["state"] = _randn(g, slots, hv, dk, dv, dtype=torch.float32, scale=0.2)
        index = torch.randperm(slots, generator=g, device="cuda")[:b].to(torch.int32)
        if case["idle"]:
            index[b - min(case["idle"], b - 1):] = -1
        st["index"] = index
        st["out"].zero_()
        st["state_out"] = st["state"].clone()
        st["live"] = [i for i in range(b) if not case["idle"] or i < b - min(case["idle"], b - 1)]
    else:
        st["state"] = _randn(g, b, hv, dk, dv, dtype=torch.float32, scale=0.2) if case["start"] else None
        st["state_out"] = torch.empty(b, hv, dk, dv, dtype=torch.float32, device="cuda")
        st["lens"] = lens
        cu = [0]
        for x in lens:
            cu.append(cu[-1] + x)
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        # where each sequence's t-th token lies (its last one behind the end), for the plain form
        at = torch.arange(max(lens), device="cuda")[None, :]
        first, count = st["cu"][:-1, None].long(), torch.tensor(lens, device="cuda")[:, None]
        st["rows"] = first + torch.minimum(at, count - 1)
        st["inside"] = at < count
        if own:
            st["workspace"] = _lib().gated_delta_workspace(n, b, hv, dk, dv)
    return st


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "mrope":
        return _prepare_mrope(case, g, seed)
    if case["op"] == "attention":
        return _prepare_attention(case, g, seed)
    return _prepare_delta(case, g, seed)


# ---- the plain forms ----------------------------------------------------------

def _axis_of(case, device):
    """The axis whose position turns frequency i."""
    half = case["rotary"] // 2
    s = _sections(case)
    i = torch.arange(half, device=device)
    if case["interleaved"]:
        axis = torch.zeros(half, dtype=torch.int64, device=device)
        for a in (1, 2):
            axis[(i % 3 == a) & (i < 3 * s[a])] = a
        return axis
    return (i >= s[0]).long() + (i >= s[0] + s[1]).long()


def _rotate(x, cos, sin, half):
    x = x.float()
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], dim=-1).to(torch.float16)


def _plain_mrope(st):
    case = st["case"]
    half, page = case["rotary"] // 2, case["page"]
    inv = _THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = st["positions"].double()[_axis_of(case, "cuda")].t() * inv
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    st["q_out"].copy_(_rotate(st["q"], cos, sin, half))
    k = _rotate(st["k"], cos, sin, half)
    index = st["index"].long()
    live = (index >= 0).nonzero()[:, 0]
    index = index[live]
    row = live if st["seq"] is None else st["seq"].long()[live]
    where = st["table"].long()[row, index // page]
    st["ck"][where, :, index % page] = k[live]
    st["cv"][where, :, index % page] = st["v"][live]
    return st["q_out"], st["ck"], st["cv"]


def _plain_attention(st):
    case = st["case"]
    b, hq, hk, d, page = case["batch"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    group = hq // hk
    # sequences in slices, so that their fp32 copies stay within a few GB
    width = st["table"].shape[1]
    step = max(1, (1 << 29) // (width * page * hk * d))
    for at in range(0, b, step):
        table = st["table"][at:at + step].long().clamp(min=0)
        n = table.shape[0]
        length = st["lengths"][at:at + n, None].long()
        seen = torch.arange(width * page, device="cuda")[None] < length
        k = st["ck"][table].transpose(2, 3).reshape(n, width * page, hk, d).float()
        v = st["cv"][table].transpose(2, 3).reshape(n, width * page, hk, d).float()
        v = v.masked_fill(~seen[:, :, None, None], 0.0)
        q = st["q"][at:at + n].float().reshape(n, hk, group, d)
        s = torch.matmul(q, k.permute(0, 2, 3, 1)) * d ** -0.5
        s = s.masked_fill(~seen[:, None, None], -math.inf)
        top = s.amax(dim=-1, keepdim=True)
        p = torch.exp(s - top.clamp(min=-1e30))
        total = p.sum(dim=-1, keepdim=True)
        o = torch.matmul(p, v.transpose(1, 2)) / total.clamp(min=1e-30)
        st["out"][at:at + n] = o.reshape(n, hq, d).to(torch.float16)
        st["lse"][at:at + n] = (top + torch.log(total)).reshape(n, hq)
    return st["out"], st["lse"]


def _unit(x):
    x = x.float()
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _plain_delta_step(st):
    case = st["case"]
    r = case["v_heads"] // case["k_heads"]
    n = len(st["live"])
    slot = st["index"][:n].long()
    q = _unit(st["q"][:n]).repeat_interleave(r, dim=1) * case["dk"] ** -0.5
    k = _unit(st["k"][:n]).repeat_interleave(r, dim=1)
    s = st["state"][slot] * torch.exp(st["g"][:n])[..., None, None]
    u = (st["v"][:n].float() - (k[..., None] * s).sum(2)) * st["beta"][:n, :, None]
    s = s + k[..., None] * u[:, :, None]
    st["out"][:n] = (q[..., None] * s).sum(2).to(torch.float16)
    st["state_out"][slot] = s
    return st["out"], st["state_out"]


def _plain_delta_prefill(st):
    case = st["case"]
    b, hv, dk, dv = case["batch"], case["v_heads"], case["dk"], case["dv"]
    r = hv // case["k_heads"]
    rows = st["rows"]
    q = (_unit(st["q"]) * dk ** -0.5).repeat_interleave(r, dim=1)[rows]
    k = _unit(st["k"]).repeat_interleave(r, dim=1)[rows]
    # behind a sequence's end nothing decays and nothing is written
    beta = (st["beta"][rows] * st["inside"][..., None])[..., None, None]
    decay = torch.exp(st["g"][rows] * st["inside"][..., None])[..., None, None]
    v = st["v"].float()[rows]
    s = torch.zeros(b, hv, dk, dv, device="cuda") if st["state"] is None else st["state"].clone()
    out = torch.empty(b, rows.shape[1], hv, dv, dtype=torch.float16, device="cuda")
    for t in range(rows.shape[1]):
        s *= decay[:, t]
        u = (v[:, t, :, None] - torch.matmul(k[:, t, :, None], s)) * beta[:, t]
        s += k[:, t, :, :, None] * u
        out[:, t] = torch.matmul(q[:, t, :, None], s)[:, :, 0].to(torch.float16)
    st["out"].copy_(out[st["inside"]])
    st["state_out"].copy_(s)
    return st["out"], st["state_out"]


def _call(st):
    """The same through the package's entry points."""
    m, op = _lib(), st["case"]["op"]
    if op == "mrope":
        m.mrope_append_kv(st["q"], st["k"], st["v"], st["positions"], st["rope"], st["cache"], st["table"],
                          st["index"], st["q_out"], seq=st["seq"])
        return st["q_out"], st["ck"], st["cv"]
    if op == "attention":
        m.paged_attention_decode(st["q"], st["cache"], st["table"], st["lengths"], st["out"], st["workspace"],
                                 lse=st["lse"])
        return st["out"], st["lse"]
    if op == "delta_step":
        m.gated_delta_step(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"], st["out"],
                           state_out=st["state_out"], index=st["index"], l2_eps=1e-6)
        return st["out"], st["state_out"]
    m.gated_delta_prefill(st["q"], st["k"], st["v"], st["g"], st["beta"], st["cu"], st["state"], st["out"],
                          st["workspace"], state_out=st["state_out"], l2_eps=1e-6)
    return st["out"], st["state_out"]


def run(st):
    if own:
        return _call(st)
    return {"mrope": _plain_mrope, "attention": _plain_attention, "delta_step": _plain_delta_step,
            "delta_prefill": _plain_delta_prefill}[st["case"]["op"]](st)


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    if case["op"] == "mrope":
        n, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
        live = n - min(case["idle"], n - 1) if case["idle"] else n
        return {"bytes": 2 * n * hq * d * 2 + 4 * live * hk * d * 2 + n * 20,
                "flops": 3 * (n * hq + live * hk) * case["rotary"]}
    if case["op"] == "attention":
        hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
        keys = sum(_lengths(case))
        return {"bytes": keys * hk * d * 4 + case["batch"] * hq * (d * 4 + 4), "flops": 4 * keys * hq * d}
    hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["dk"], case["dv"]
    if case["op"] == "delta_step":
        n = b = case["batch"] - (min(case["idle"], case["batch"] - 1) if case["idle"] else 0)
        reads = 1
    else:
        n, b = sum(_lengths(case)), case["batch"]
        reads = 1 if case["start"] else 0
    return {"bytes": n * (4 * hk * dk + 4 * hv * dv + 8 * hv) + (1 + reads) * b * hv * dk * dv * 4,
            "flops": 7 * n * hv * dk * dv}


# ---- the definitions in 64 bits ---------------------------------------------------

def _exact_mrope(case, st):
    half, page, d = case["rotary"] // 2, case["page"], case["dim"]
    sec = _sections(case)
    turn = torch.empty(case["tokens"], half, dtype=torch.complex128, device="cuda")
    pos = st["positions"].double()
    for i in range(half):
        if case["interleaved"]:
            axis = i % 3 if i % 3 and i < 3 * sec[i % 3] else 0
        else:
            axis = 0 if i < sec[0] else 1 if i < sec[0] + sec[1] else 2
        a = pos[axis] * math.exp(-math.log(_THETA) * i / half)
        turn[:, i] = torch.polar(torch.ones_like(a), a)

    def turned(x):
        y = x.double().clone()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn[:, None]
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
        return y

    q, k = turned(st["q"]), turned(st["k"])
    ck, cv = st["ck"].double(), st["cv"].double()
    index, table = st["index"].tolist(), st["table"].tolist()
    for t, i in enumerate(index):
        if i >= 0:
            p = table[t if st["seq"] is None else 0][i // page]
            ck[p, :, i % page] = k[t]
            cv[p, :, i % page] = st["v"][t].double()
    return q, ck, cv


def _exact_attention(case, st):
    b, hq, hk, d = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, hq), -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        used = st["table"][i, :(n + case["page"] - 1) // case["page"]].long()
        for h in range(hk):
            k = st["ck"][used, h].reshape(-1, d)[:n].double()
            v = st["cv"][used, h].reshape(-1, d)[:n].double()
            rows = slice(h * (hq // hk), (h + 1) * (hq // hk))
            s = st["q"][i, rows].double() @ k.t() / math.sqrt(d)
            lse[i, rows] = torch.logsumexp(s, dim=1)
            out[i, rows] = torch.softmax(s, dim=1) @ v
    return out, lse


def _exact_delta(case, st):
    hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["dk"], case["dv"]
    step = case["op"] == "delta_step"
    head = torch.arange(hv, device="cuda") // (hv // hk)

    def unit(x):
        x = x.double()
        return (x * torch.rsqrt(torch.einsum("thd,thd->th", x, x) + 1e-6)[..., None])[:, head]

    q, k, v = unit(st["q"]) / math.sqrt(dk), unit(st["k"]), st["v"].double()
    keep, beta = torch.exp(st["g"].double()), st["beta"].double()
    out = torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    if step:
        final = st["state_out"].double()
        for t in st["live"]:
            slot = int(st["index"][t])
            s = st["state"][slot].double() * keep[t, :, None, None]
            s += torch.einsum("hk,hv->hkv", k[t], beta[t, :, None] * (v[t] - torch.einsum("hk,hkv->hv", k[t], s)))
            out[t], final[slot] = torch.einsum("hk,hkv->hv", q[t], s), s
        return out, final
    final = torch.zeros(case["batch"], hv, dk, dv, dtype=torch.float64, device="cuda")
    if st["state"] is not None:
        final += st["state"].double()
    first = 0
    # blocks of tokens: with S the state before a block and c_t the decay up to token t, the written
    # rows u solve (I + L) u = beta (v - c k S), L_ts = beta_t (c_t / c_s) k_t.k_s below the diagonal
    for i, n in enumerate(st["lens"]):
        for lo in range(first, first + n, 32):
            rows = slice(lo, min(lo + 32, first + n))
            s, kk, qq, vv = final[i], k[rows].transpose(0, 1), q[rows].transpose(0, 1), v[rows].transpose(0, 1)
            c = torch.cumsum(st["g"][rows].double(), 0).t()
            ratio = torch.exp((c[:, :, None] - c[:, None, :]).tril()).tril()
            bb = beta[rows].t()[..., None]
            low = (bb * ratio * (kk @ kk.transpose(1, 2))).tril(-1)
            eye = torch.eye(low.shape[1], dtype=torch.float64, device="cuda")
            u = torch.linalg.solve_triangular(eye + low, bb * (vv - torch.exp(c)[..., None] * (kk @ s)), upper=False)
            out[rows] = (torch.exp(c)[..., None] * (qq @ s) + (ratio * (qq @ kk.transpose(1, 2))) @ u).transpose(0, 1)
            last = torch.exp(c[:, -1:] - c)[..., None]
            final[i] = torch.exp(c[:, -1])[:, None, None] * s + (last * kk).transpose(1, 2) @ u
        first += n
    return out, final


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "mrope":
        return _exact_mrope(case, st)
    if case["op"] == "attention":
        return _exact_attention(case, st)
    return _exact_delta(case, st)
