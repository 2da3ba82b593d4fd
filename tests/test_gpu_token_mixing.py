"""The token-mixing operators on the GPU - rotary positions with cache append,
paged decode attention, the gated delta rule - against plain fp64
computations.

Tolerances.  An fp16 output may be off by its rounding, 2^-11 of its value
(2^-25 where it is subnormal), plus what fp32 arithmetic leaves:
 * rope: the angle is exact to 2^-24 of a half turn and sin, cos to a few
   2^-24, so 2^-20 (|a| + |b|) covers angle, functions and the two products;
 * attention: fp32 scores of D products, error at most D 2^-24 sum|q k| scale =
   e; exp turns it into a relative 2 e of the probabilities; P is kept to 2^-22;
 * delta: one token's products of DK terms are off by (DK + 8) 2^-24 of the
   column norms, and since I - beta k k^T and the decay never enlarge a column
   (|k| <= 1, beta <= 1, g <= 0), T tokens add up to T times that.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_ULP16 = 2.0 ** -11
SUB16 = 2.0 ** -25


def close16(got, ref, extra, what):
    import torch
    assert torch.isfinite(got).all(), what
    err = (got.double() - ref).abs()
    bound = HALF_ULP16 * ref.abs() + SUB16 + extra
    worst = (err / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound, max error {err.max().item():.3g}"


def gen(seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=None, scale=1.0):
    import torch
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype or torch.float16)


# ---- rope ---------------------------------------------------------------------

def rope_ref(x, positions, sections, interleaved, theta, rotary):
    """fp64, frequency by frequency."""
    import torch
    half, n_axes = rotary // 2, len(sections)
    y = x.double().clone()
    for i in range(half):
        if interleaved:
            axis = i % n_axes if i % n_axes and i < n_axes * sections[i % n_axes] else 0
        else:
            axis = next(a for a in range(n_axes) if i < sum(sections[:a + 1]))
        ang = positions[axis].double() * theta ** (-2.0 * i / rotary)
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        a, b = x[..., i].double(), x[..., i + half].double()
        y[..., i], y[..., i + half] = a * c - b * s, b * c + a * s
    return y


def rope_extra(x, rotary):
    import torch
    half = rotary // 2
    e = torch.zeros_like(x, dtype=torch.float64)
    both = x[..., :half].double().abs() + x[..., half:rotary].double().abs()
    e[..., :half] = e[..., half:rotary] = both * 2.0 ** -20
    return e


@pytest.mark.parametrize("tokens,heads,dim,rotary,sections,interleaved", [
    (1, 8, 256, 64, [12, 10, 10], True), (7, 3, 64, 64, [32], False), (1300, 2, 128, 32, [8, 4, 4], False),
    (5, 1, 256, 256, [48, 40, 40], True), (3, 5, 24, 16, [2, 2, 2, 2], True), (2, 4, 80, 48, [0, 24], False)])
def test_mrope(cuda, tokens, heads, dim, rotary, sections, interleaved):
    import mcv_b200 as mcv
    torch = cuda
    g = gen(tokens + dim)
    x = randn(g, tokens, heads, dim)
    pos = torch.randint(0, 1 << 20, (len(sections), tokens), generator=g, device="cuda", dtype=torch.int32)
    rope = mcv.MRope(rotary, sections, interleaved, 1.0e7)
    out = torch.empty_like(x)
    mcv.mrope(x, pos, rope, out)
    ref = rope_ref(x, pos, sections, interleaved, 1.0e7, rotary)
    close16(out, ref, rope_extra(x, rotary), "mrope")
    assert torch.equal(out[..., rotary:], x[..., rotary:])
    # in place, in a wider row and with the heads first
    for wide in (torch.zeros(tokens, heads, 2 * dim, dtype=torch.float16, device="cuda")[:, :, dim:],
                 torch.zeros(heads, tokens, dim, dtype=torch.float16, device="cuda").transpose(0, 1)):
        wide.copy_(x)
        mcv.mrope(wide, pos, rope, wide)
        assert torch.equal(wide, out)


@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,page", [(1, 8, 2, 256, 64, 16), (33, 4, 4, 64, 32, 7),
                                                          (2000, 6, 1, 128, 128, 24), (9, 2, 2, 256, 64, 1),
                                                          (700, 72, 20, 256, 64, 16), (50, 40, 33, 64, 64, 8),
                                                          (1500, 12, 3, 80, 48, 16), (3, 2, 1, 512, 256, 4)])
def test_mrope_append_kv(cuda, tokens, hq, hk, dim, rotary, page):
    """Scattered tokens of several sequences, some not written; slots that no
    token has stay as they were."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(tokens * 3 + page)
    fused = randn(g, tokens, (hq + 2 * hk) * dim)
    q = fused[:, :hq * dim].unflatten(1, (hq, dim))
    k = fused[:, hq * dim:(hq + hk) * dim].unflatten(1, (hk, dim))
    v = fused[:, (hq + hk) * dim:].unflatten(1, (hk, dim))
    half = rotary // 2
    sections = [half - 2 * (half // 3), half // 3, half // 3]
    pos = torch.randint(0, 300000, (3, tokens), generator=g, device="cuda", dtype=torch.int32)
    rows = 5
    per_row = -(-tokens // rows)
    cols = -(-per_row // page) + 1
    table = torch.randperm(rows * cols + 2, generator=g, device="cuda")[:rows * cols].reshape(rows, cols).int()
    order = torch.randperm(tokens, generator=g, device="cuda")
    seq, index = (order % rows).int(), (order // rows).int()
    index[order % 4 == 3] = -1
    both = randn(g, rows * cols + 2, 2, hk, page, dim)
    cache = mcv.PagedKVCache(both[:, 0], both[:, 1])   # k and v pages alternate in one buffer
    want = both.clone()
    q_out = torch.empty(tokens, hq, dim, dtype=torch.float16, device="cuda")
    mcv.device_errors()
    mcv.mrope_append_kv(q, k, v, pos, mcv.MRope(rotary, sections, True), cache, table, index, q_out, seq=seq)
    assert mcv.device_errors() == 0
    close16(q_out, rope_ref(q, pos, sections, True, 1.0e7, rotary), rope_extra(q, rotary), "q")
    kref, kx = rope_ref(k, pos, sections, True, 1.0e7, rotary), rope_extra(k, rotary)
    live = (index >= 0).nonzero()[:, 0]
    i = index[live].long()
    p = table.long()[seq[live].long(), i // page]
    close16(both[p, 0, :, i % page], kref[live], kx[live], "k")
    want[p, 0, :, i % page] = both[p, 0, :, i % page]
    want[p, 1, :, i % page] = v[live]
    assert torch.equal(both, want)


def test_mrope_append_bad_indices(cuda):
    """Rows, places and pages out of range are not followed and are reported."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(5)
    q, k, v = (randn(g, 6, 2, 64) for _ in range(3))
    cache = mcv.PagedKVCache(torch.zeros(3, 2, 4, 64, dtype=torch.float16, device="cuda"),
                             torch.zeros(3, 2, 4, 64, dtype=torch.float16, device="cuda"))
    pos = torch.arange(6, dtype=torch.int32, device="cuda")[None].contiguous()
    table = torch.tensor([[0, 3], [-1, 2]], dtype=torch.int32, device="cuda")
    seq = torch.tensor([0, 0, 1, 2, -1, 1], dtype=torch.int32, device="cuda")
    index = torch.tensor([1, 5, 0, 0, 0, 8], dtype=torch.int32, device="cuda")
    q_out = torch.empty_like(q)
    mcv.device_errors()
    mcv.mrope_append_kv(q, k, v, pos, mcv.MRope(64, [32]), cache, table, index, q_out, seq=seq)
    assert mcv.device_errors() == 2
    assert torch.equal(cache.v[0, :, 1], v[0])
    cache.v[0, :, 1] = 0
    assert not cache.v.any()
    assert torch.isfinite(q_out).all()


# ---- attention ------------------------------------------------------------------

def attention_setup(torch, g, lens, hq, hk, dim, page, qscale=1.5, spare=3, poison=True):
    """Sequences on scattered pages; every slot without a key holds NaN."""
    need = [-(-max(0, n) // page) for n in lens]
    cols, pages = max(1, max(need)) + 1, sum(need) + spare
    perm = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), cols), 1 << 30, dtype=torch.int32, device="cuda")
    ck, cv = (torch.full((pages, hk, page, dim), math.nan if poison else 0.0, dtype=torch.float16, device="cuda")
              for _ in range(2))
    keys = []
    at = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = perm[at:at + need[b]]
        kk, vv = randn(g, max(n, 0), hk, dim), randn(g, max(n, 0), hk, dim)
        i = torch.arange(max(n, 0), device="cuda")
        p = table[b].long()[i // page]
        ck[p, :, i % page], cv[p, :, i % page] = kk, vv
        keys.append((kk, vv))
        at += need[b]
    q = randn(g, len(lens), hq, dim, scale=qscale)
    return q, ck, cv, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), keys


def attention_check(torch, q, keys, scale, out, lse, what):
    group = q.shape[1] // keys[0][0].shape[1]
    for b, (k, v) in enumerate(keys):
        if k.shape[0] == 0:
            assert not out[b].any() and (lse[b] == -math.inf).all(), what
            continue
        kk, vv = (x.double().repeat_interleave(group, dim=1).transpose(0, 1) for x in (k, v))
        s = torch.einsum("hd,hnd->hn", q[b].double(), kk) * scale
        e = torch.einsum("hd,hnd->hn", q[b].double().abs(), kk.abs()).amax(1) * scale * q.shape[2] * 2.0 ** -24
        ref = torch.einsum("hn,hnd->hd", torch.softmax(s, 1), vv)
        spread = torch.einsum("hn,hnd->hd", torch.softmax(s, 1), vv.abs())
        close16(out[b], ref, spread * (2 * e[:, None] + 2.0 ** -18), f"{what} row {b}")
        ref_lse = torch.logsumexp(s, 1)
        assert ((lse[b].double() - ref_lse).abs() <= 2 * e + 2.0 ** -20 * (1 + ref_lse.abs())).all(), what


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,hq,hk,page", [
    ([1], 8, 2, 16), ([15, 16, 17, 0, 1, 33], 4, 4, 16), ([611], 8, 2, 16), ([7, 0, 300, 64, 5], 10, 2, 7),
    ([129, 1000], 16, 1, 24), ([40, 2], 17, 1, 1), ([513], 36, 2, 64), ([0, 0], 2, 1, 16), ([-3, 20], 6, 3, 32)])
def test_attention(cuda, dim, lens, hq, hk, page):
    import mcv_b200 as mcv
    torch = cuda
    g = gen(dim + sum(lens) + hq)
    q, ck, cv, table, lengths, keys = attention_setup(torch, g, lens, hq, hk, dim, page)
    ws = mcv.paged_attention_workspace(len(lens), hq, hk, dim)
    out = torch.full((len(lens), hq, dim), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((len(lens), hq), 7.0, device="cuda")
    cache = mcv.PagedKVCache(ck, cv)
    mcv.device_errors()
    mcv.paged_attention_decode(q, cache, table, lengths, out, ws, lse=lse)
    attention_check(torch, q, keys, dim ** -0.5, out, lse, f"attention {lens}")
    # again on the same workspace: the same bits, with and without lse, with a scale, from a wider row
    wide = torch.zeros(len(lens), hq, 2 * dim, dtype=torch.float16, device="cuda")
    wide[:, :, :dim] = q
    again = torch.empty_like(out)
    mcv.paged_attention_decode(wide[:, :, :dim], cache, table, lengths, again, ws, scale=dim ** -0.5)
    assert torch.equal(out, again)
    assert mcv.device_errors() == 0


@pytest.mark.parametrize("dim,hq,hk,page,batch,longest", [(256, 8, 2, 16, 1, 20011), (256, 16, 2, 48, 3, 9001),
                                                          (128, 32, 8, 16, 70, 900), (64, 8, 8, 32, 300, 90),
                                                          (64, 12, 4, 16, 4096, 12)])
def test_attention_long_and_ragged(cuda, dim, hq, hk, page, batch, longest):
    """Rows cut over many blocks, blocks with many rows, results joined twice."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(batch + longest)
    r = np.random.default_rng(batch)
    lens = [longest] + [int(x) for x in r.integers(0, longest + 1, batch - 1)]
    q, ck, cv, table, lengths, keys = attention_setup(torch, g, lens, hq, hk, dim, page)
    ws = mcv.paged_attention_workspace(batch, hq, hk, dim)
    out = torch.empty(batch, hq, dim, dtype=torch.float16, device="cuda")
    lse = torch.empty(batch, hq, device="cuda")
    cache = mcv.PagedKVCache(ck, cv)
    mcv.paged_attention_decode(q, cache, table, lengths, out, ws, lse=lse)
    some = range(batch) if batch <= 70 else [int(x) for x in r.integers(0, batch, 60)]
    sel = torch.tensor(list(some), device="cuda")
    attention_check(torch, q[sel], [keys[i] for i in some], dim ** -0.5, out[sel], lse[sel], "ragged")
    for _ in range(5):
        again = torch.empty_like(out)
        mcv.paged_attention_decode(q, cache, table, lengths, again, ws)
        assert torch.equal(out, again)


def test_attention_extreme_scores(cuda):
    """Very large scores either way, keys whose weight underflows, equal scores."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(3)
    q, ck, cv, table, lengths, keys = attention_setup(torch, g, [200, 200, 64], 8, 2, 64, 16)
    q[0] *= 200.0
    q[1] = 0.0
    i = torch.arange(200, device="cuda")
    p = table[0].long()[i // 16]
    ck[p, :, i % 16] = keys[0][0] * 20
    keys[0] = (keys[0][0] * 20, keys[0][1])
    out, lse = torch.empty_like(q), torch.empty(3, 8, device="cuda")
    ws = mcv.paged_attention_workspace(3, 8, 2, 64)
    mcv.paged_attention_decode(q, mcv.PagedKVCache(ck, cv), table, lengths, out, ws, lse=lse)
    attention_check(torch, q, keys, 0.125, out, lse, "extreme")


def test_attention_workspace_shared_by_shapes(cuda):
    """One workspace, large enough for each, serves calls of different heads."""
    import mcv_b200 as mcv
    torch = cuda
    shapes = [(64, 8, 8, 5000), (256, 16, 2, 5000), (64, 32, 2, 900), (128, 8, 1, 7001), (64, 8, 8, 5000)]
    ws = max((mcv.paged_attention_workspace(1, hq, hk, d) for d, hq, hk, _ in shapes), key=lambda w: w.numel())
    for d, hq, hk, n in shapes:
        g = gen(d + n)
        q, ck, cv, table, lengths, keys = attention_setup(torch, g, [n, n // 3], hq, hk, d, 16)
        out, lse = torch.empty_like(q), torch.empty(2, hq, device="cuda")
        mcv.paged_attention_decode(q, mcv.PagedKVCache(ck, cv), table, lengths, out, ws, lse=lse)
        attention_check(torch, q, keys, d ** -0.5, out, lse, "shared workspace")


def test_attention_bad_pages_and_lengths(cuda):
    """A page out of range reads as zeros, a length beyond the table is cut;
    both are reported, and other rows are untouched by it."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(9)
    q, ck, cv, table, lengths, keys = attention_setup(torch, g, [40, 48, 50], 4, 2, 64, 16)
    table[0, 1] = ck.shape[0]
    table[1, 0] = -1
    lengths[2] = 1 << 30
    table[2, 4:] = table[2, 0]
    full = int(table.shape[1]) * 16
    ws = mcv.paged_attention_workspace(3, 4, 2, 64)
    out = torch.empty_like(q)
    ck, cv = torch.nan_to_num(ck, nan=0.5), torch.nan_to_num(cv, nan=0.25)
    mcv.device_errors()
    mcv.paged_attention_decode(q, mcv.PagedKVCache(ck, cv), table, lengths, out, ws)
    assert mcv.device_errors() == 2
    z = torch.zeros(16, 2, 64, dtype=torch.float16, device="cuda")
    k0, v0 = keys[0]
    k1, v1 = keys[1]
    i = torch.arange(full, device="cuda")
    p = table[2].long()[i // 16]
    ok = [(torch.cat([k0[:16], z, k0[32:]]), torch.cat([v0[:16], z, v0[32:]])),
          (torch.cat([z, k1[16:]]), torch.cat([z, v1[16:]])), (ck[p, :, i % 16], cv[p, :, i % 16])]
    lse = torch.empty(3, 4, device="cuda")
    mcv.paged_attention_decode(q, mcv.PagedKVCache(ck, cv), table, lengths, out, ws, lse=lse)
    attention_check(torch, q, ok, 0.125, out, lse, "bad pages")
    mcv.device_errors()


def test_attention_far_pages(cuda):
    """Pages whose elements lie beyond 2^31."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(11)
    base = torch.empty((1 << 32) + (1 << 20), dtype=torch.float16, device="cuda")
    view = lambda off: base.as_strided((5, 2, 16, 64), (1 << 30, 16 * 64, 64, 1), off)
    ck, cv = view(0), view(1 << 16)
    table = torch.tensor([[4, 0, 3]], dtype=torch.int32, device="cuda")
    k, v, q = randn(g, 37, 2, 64), randn(g, 37, 2, 64), randn(g, 37, 4, 64)
    cache = mcv.PagedKVCache(ck, cv)
    idx = torch.arange(37, dtype=torch.int32, device="cuda")
    qo = torch.empty_like(q)
    zero = torch.zeros(1, 37, dtype=torch.int32, device="cuda")
    mcv.mrope_append_kv(q, k, v, zero, mcv.MRope(64, [32]), cache, table, idx, qo, seq=torch.zeros_like(idx))
    assert torch.equal(qo, q)
    out, lse = torch.empty(1, 4, 64, dtype=torch.float16, device="cuda"), torch.empty(1, 4, device="cuda")
    mcv.paged_attention_decode(q[:1], cache, table, torch.tensor([37], dtype=torch.int32, device="cuda"), out,
                               mcv.paged_attention_workspace(1, 4, 2, 64), lse=lse)
    attention_check(torch, q[:1], [(k, v)], 0.125, out, lse, "far pages")


# ---- the gated delta rule -----------------------------------------------------------

def delta_inputs(torch, g, n, hk, hv, dk, dv, decay=0.3):
    fused = randn(g, n, 2 * hk * dk + hv * dv)
    q = fused[:, :hk * dk].unflatten(1, (hk, dk))
    k = fused[:, hk * dk:2 * hk * dk].unflatten(1, (hk, dk))
    v = fused[:, 2 * hk * dk:].unflatten(1, (hv, dv))
    gl = -torch.rand(n, hv, generator=g, device="cuda") * decay
    beta = torch.rand(n, hv, generator=g, device="cuda")
    return q, k, v, gl, beta


def delta_ref(torch, q, k, v, g, beta, s, scale, l2_eps):
    """Token by token in fp64; also the largest column size seen."""
    r = v.shape[1] // q.shape[1]

    def prep(x):
        x = x.double()
        if l2_eps is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) + l2_eps)
        return x.repeat_interleave(r, dim=1)

    q, k, v = prep(q), prep(k), v.double()
    s = s.double().clone()
    out = torch.empty(v.shape, dtype=torch.float64, device="cuda")
    size = s.norm(dim=1)
    for t in range(v.shape[0]):
        s = s * torch.exp(g[t].double())[:, None, None]
        u = beta[t].double()[:, None] * (v[t] - torch.einsum("hkv,hk->hv", s, k[t]))
        s = s + k[t][:, :, None] * u[:, None]
        out[t] = torch.einsum("hkv,hk->hv", s, q[t]) * scale
        size = torch.maximum(size, s.norm(dim=1) + v[t].abs())
    return out, s, size


def delta_check(torch, args, state, out, state_out, scale, l2_eps, what):
    q, k, v, g, beta = args
    ref, s, size = delta_ref(torch, q, k, v, g, beta, state, scale, l2_eps)
    dk = q.shape[2]
    fp32 = (len(v) + 1) * (dk + 8) * 2.0 ** -24 * size      # [heads, dv], per column
    if l2_eps is None:
        qn = q.double().norm(dim=2).repeat_interleave(v.shape[1] // q.shape[1], dim=1)[..., None]
    else:
        qn = 1.0
    close16(out, ref, 2 * fp32[None] * qn * abs(scale), what)
    if state_out is not None:
        worst = ((state_out.double() - s).abs() / (fp32[:, None] + 2.0 ** -24 * s.abs())).max().item()
        assert worst <= 1.0, f"{what}: state at {worst:.3f} of the bound"


@pytest.mark.parametrize("batch,hk,hv,dk,dv", [(1, 16, 16, 128, 128), (5, 2, 4, 64, 48), (40, 4, 8, 128, 64),
                                               (3, 1, 3, 64, 272), (2, 3, 3, 128, 16)])
@pytest.mark.parametrize("l2_eps", [1e-6, None])
def test_delta_step(cuda, batch, hk, hv, dk, dv, l2_eps):
    import mcv_b200 as mcv
    torch = cuda
    g = gen(batch + dv)
    q, k, v, gl, beta = delta_inputs(torch, g, batch, hk, hv, dk, dv)
    if l2_eps is None:
        q, k = q / 16, k / 16
    slots = batch + 3
    state = randn(g, slots, hv, dk, dv, dtype=torch.float32)
    index = torch.randperm(slots, generator=g, device="cuda")[:batch].int()
    if batch > 2:
        index[1] = -1
    out = torch.full((batch, hv, dv), 3.0, dtype=torch.float16, device="cuda")
    new = state.clone()
    mcv.gated_delta_step(q, k, v, gl, beta, state, out, state_out=new, index=index, l2_eps=l2_eps)
    used = []
    for b in range(batch):
        i = int(index[b])
        if i < 0:
            assert (out[b] == 3.0).all()
            continue
        used.append(i)
        delta_check(torch, [x[b:b + 1] for x in (q, k, v, gl, beta)], state[i], out[b:b + 1], new[i], dk ** -0.5, l2_eps,
                    f"step {b}")
    rest = [i for i in range(slots) if i not in used]
    assert torch.equal(new[rest], state[rest])
    # in place, the same bits
    inplace, out2 = state.clone(), torch.full_like(out, 3.0)
    mcv.gated_delta_step(q, k, v, gl, beta, inplace, out2, index=index, l2_eps=l2_eps)
    assert torch.equal(inplace, new) and torch.equal(out, out2)


@pytest.mark.parametrize("lens,hk,hv,dk,dv", [
    ([1], 2, 2, 128, 128), ([61], 4, 4, 128, 128), ([64], 1, 2, 64, 64), ([65, 0, 1, 128, 200], 2, 4, 128, 64),
    ([300, 5], 1, 1, 64, 48), ([700], 2, 2, 128, 128), ([3] * 40, 1, 1, 128, 32), ([130, 257], 1, 3, 128, 272)])
@pytest.mark.parametrize("start", [False, True])
def test_delta_prefill(cuda, lens, hk, hv, dk, dv, start):
    import mcv_b200 as mcv
    torch = cuda
    g = gen(sum(lens) + dv + start)
    b, n = len(lens), sum(lens)
    spare = 5        # rows behind the last sequence
    args = delta_inputs(torch, g, n + spare, hk, hv, dk, dv)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    slots = b + 2
    state = randn(g, slots, hv, dk, dv, dtype=torch.float32) if start else None
    index = torch.randperm(slots, generator=g, device="cuda")[:b].int() if start else None
    new = torch.full((slots if start else b, hv, dk, dv), 9.0, device="cuda")
    out = torch.full((n + spare, hv, dv), 3.0, dtype=torch.float16, device="cuda")
    ws = mcv.gated_delta_workspace(n + spare, b, hv, dk, dv)
    ws.fill_(255)      # whatever it holds
    mcv.device_errors()
    mcv.gated_delta_prefill(*args, cu, state, out, ws, state_out=new, index=index, l2_eps=1e-6)
    assert mcv.device_errors() == 0
    assert (out[n:] == 3.0).all()
    at = 0
    for i, ln in enumerate(lens):
        slot = int(index[i]) if start else i
        s0 = state[slot] if start else torch.zeros(hv, dk, dv, device="cuda")
        if ln == 0:
            assert torch.equal(new[slot], s0)
        else:
            delta_check(torch, [x[at:at + ln] for x in args], s0, out[at:at + ln], new[slot], dk ** -0.5, 1e-6,
                        f"prefill {i}")
        at += ln
    # final states dropped; in place
    out2 = torch.full_like(out, 3.0)
    if start:
        inplace = state.clone()
        mcv.gated_delta_prefill(*args, cu, inplace, out2, ws, index=index, l2_eps=1e-6)
        assert torch.equal(inplace[index.long()], new[index.long()])
    else:
        mcv.gated_delta_prefill(*args, cu, None, out2, ws, l2_eps=1e-6)
    assert torch.equal(out, out2)


@pytest.mark.parametrize("lens,hk,hv,dk,dv", [
    ([130, 64, 1, 0, 257], 8, 16, 128, 128), ([65] * 12, 8, 16, 64, 64), ([200, 70], 48, 48, 64, 144),
    ([449, 321], 24, 48, 128, 16), ([100] * 40, 2, 4, 128, 96)])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -9, 2.0 ** 7])
def test_delta_prefill_many_heads(cuda, lens, hk, hv, dk, dv, scale):
    """Enough heads for the walk that takes whole ones; values and states of
    very different sizes from head to head and within a sequence."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(sum(lens) + dv)
    b, n = len(lens), sum(lens)
    q, k, v, gl, beta = delta_inputs(torch, g, n, hk, hv, dk, dv)
    v = v * (scale * 2.0 ** torch.randint(-6, 6, (1, hv, 1), generator=g, device="cuda").float()).half()
    v[n // 2:] *= 0.125
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    index = torch.randperm(b + 1, generator=g, device="cuda")[:b].int()
    state = randn(g, b + 1, hv, dk, dv, dtype=torch.float32) * scale
    new, out = torch.full_like(state, 9.0), torch.empty(n, hv, dv, dtype=torch.float16, device="cuda")
    ws = mcv.gated_delta_workspace(n, b, hv, dk, dv)
    ws.fill_(255)
    mcv.device_errors()
    mcv.gated_delta_prefill(q, k, v, gl, beta, cu, state, out, ws, state_out=new, index=index, l2_eps=1e-6)
    assert mcv.device_errors() == 0
    at = 0
    for i, ln in enumerate(lens):
        slot = int(index[i])
        if ln == 0:
            assert torch.equal(new[slot], state[slot])
        else:
            delta_check(torch, [x[at:at + ln] for x in (q, k, v, gl, beta)], state[slot], out[at:at + ln], new[slot], dk ** -0.5,
                        1e-6, f"sequence {i}")
        at += ln
    # in place, without a state at the start, and as given keys and queries
    inplace, out2 = state.clone(), torch.empty_like(out)
    mcv.gated_delta_prefill(q, k, v, gl, beta, cu, inplace, out2, ws, index=index, l2_eps=1e-6)
    assert torch.equal(out, out2) and torch.equal(inplace[index.long()], new[index.long()])
    kn, qs = (k / 16).contiguous(), (q * 3).contiguous()
    first = torch.empty(b, hv, dk, dv, device="cuda")
    mcv.gated_delta_prefill(qs, kn, v, gl, beta, cu, None, out2, ws, state_out=first, scale=0.5)
    zero = torch.zeros(hv, dk, dv, device="cuda")
    delta_check(torch, [x[:lens[0]] for x in (qs, kn, v, gl, beta)], zero, out2[:lens[0]], first[0], 0.5, None, "as given")


@pytest.mark.parametrize("kind", ["forget", "keep", "write", "none", "mixed"])
def test_delta_prefill_gates(cuda, kind):
    """Decays that erase everything (also -inf), none at all, full and no
    writing, the same key again and again."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(77)
    n, h = 200, 2
    q, k, v, gl, beta = delta_inputs(torch, g, n, h, h, 128, 128)
    if kind == "forget":
        gl[::7] = -300.0
        gl[50] = -math.inf
    elif kind == "keep":
        gl.zero_()
    elif kind == "write":
        beta.fill_(1.0)
        k = k[:1].expand(n, h, 128).contiguous()
        gl.zero_()
    elif kind == "none":
        beta.zero_()
    else:
        gl = gl * torch.randint(0, 2, gl.shape, generator=g, device="cuda") * 40
    state = randn(g, 1, h, 128, 128, dtype=torch.float32)
    out, new = torch.empty(n, h, 128, dtype=torch.float16, device="cuda"), torch.empty_like(state)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    mcv.gated_delta_prefill(q, k, v, gl, beta, cu, state, out, mcv.gated_delta_workspace(n, 1, h, 128, 128),
                            state_out=new, l2_eps=1e-6)
    delta_check(torch, (q, k, v, gl, beta), state[0], out, new[0], 128 ** -0.5, 1e-6, kind)


def test_delta_prefill_neighbours_do_not_mix(cuda):
    """A sequence of NaN between two others leaves them alone, and sequence
    bounds or slots out of range are reported and not followed."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(78)
    lens = [70, 33, 90]
    args = delta_inputs(torch, g, sum(lens), 2, 2, 128, 128)
    for x in args[:3]:
        x[70:103] = math.nan
    cu = torch.tensor([0, 70, 103, 193], dtype=torch.int32, device="cuda")
    out = torch.empty(193, 2, 128, dtype=torch.float16, device="cuda")
    new = torch.empty(3, 2, 128, 128, device="cuda")
    ws = mcv.gated_delta_workspace(193, 3, 2, 128, 128)
    mcv.gated_delta_prefill(*args, cu, None, out, ws, state_out=new, l2_eps=1e-6)
    zero = torch.zeros(2, 128, 128, device="cuda")
    for i, (lo, hi) in enumerate([(0, 70), (103, 193)]):
        delta_check(torch, [x[lo:hi] for x in args], zero, out[lo:hi], new[2 * i], 128 ** -0.5, 1e-6, "neighbour")
    assert torch.isnan(out[70:103]).all()
    mcv.device_errors()
    new.fill_(5.0)
    out.fill_(5.0)
    bad = torch.tensor([0, 70, 60, 1000], dtype=torch.int32, device="cuda")
    mcv.gated_delta_prefill(*args, bad, None, out, ws, state_out=new, l2_eps=1e-6)
    assert mcv.device_errors() == 2
    assert (new[1:] == 5.0).all() and (out[70:] == 5.0).all()
    delta_check(torch, [x[:70] for x in args], zero, out[:70], new[0], 128 ** -0.5, 1e-6, "good sequence")
    mcv.gated_delta_prefill(*args, cu, None, out, ws, state_out=new, l2_eps=1e-6,
                            index=torch.tensor([3, -1, 0], dtype=torch.int32, device="cuda"))
    assert mcv.device_errors() == 2


# ---- together --------------------------------------------------------------------

def test_layers_of_a_conversation(cuda):
    """A full-attention and a linear layer as a conversation uses them: a prompt
    with an image into the cache and the state, then tokens one at a time from a
    captured graph on its own stream, each against the whole history."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(100)
    hq, hk, dim, rotary, page, prompt, steps = 8, 2, 256, 64, 16, 150, 9
    total = prompt + steps
    sections = [12, 10, 10]
    q, k, v = randn(g, total, hq, dim), randn(g, total, hk, dim), randn(g, total, hk, dim)
    pos = torch.arange(total, dtype=torch.int32, device="cuda").repeat(3, 1)
    pos[0, 20:120], pos[1, 20:120], pos[2, 20:120] = 20, 20 + torch.arange(100, device="cuda").int() // 10, \
        20 + torch.arange(100, device="cuda").int() % 10
    pos[:, 120:] = torch.arange(30, 30 + total - 120, device="cuda").int()
    rope = mcv.MRope(rotary, sections, True)
    cols = -(-total // page)
    cache = mcv.PagedKVCache.empty(cols + 2, hk, page, dim)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    table = torch.randperm(cols + 2, generator=g, device="cuda")[:cols].int()[None].contiguous()
    dargs = delta_inputs(torch, g, total, 4, 4, 128, 128)
    state = torch.empty(1, 4, 128, 128, device="cuda")
    dout = torch.empty(prompt, 4, 128, dtype=torch.float16, device="cuda")
    idx = torch.arange(total, dtype=torch.int32, device="cuda")
    qo = torch.empty(prompt, hq, dim, dtype=torch.float16, device="cuda")
    mcv.mrope_append_kv(q[:prompt], k[:prompt], v[:prompt], pos[:, :prompt].contiguous(), rope, cache, table,
                        idx[:prompt], qo, seq=torch.zeros(prompt, dtype=torch.int32, device="cuda"))
    mcv.gated_delta_prefill(*[x[:prompt] for x in dargs], torch.tensor([0, prompt], dtype=torch.int32, device="cuda"),
                            None, dout, mcv.gated_delta_workspace(prompt, 1, 4, 128, 128), state_out=state, l2_eps=1e-6)

    # one step on fixed buffers, captured
    bufs = [x[prompt:prompt + 1].clone() for x in (q, k, v)]
    dbufs = [x[prompt:prompt + 1].clone() for x in dargs]
    p1, i1 = pos[:, prompt:prompt + 1].contiguous(), idx[prompt:prompt + 1].clone()
    length = (i1 + 1).int()
    qr, att = torch.empty(1, hq, dim, dtype=torch.float16, device="cuda"), torch.empty(1, hq, dim, dtype=torch.float16,
                                                                                      device="cuda")
    lse, d1 = torch.empty(1, hq, device="cuda"), torch.empty(1, 4, 128, dtype=torch.float16, device="cuda")
    ws = mcv.paged_attention_workspace(1, hq, hk, dim)
    side = torch.cuda.Stream()

    def step():
        mcv.mrope_append_kv(*bufs, p1, rope, cache, table, i1, qr)
        mcv.paged_attention_decode(qr, cache, table, length, att, ws, lse=lse)
        mcv.gated_delta_step(*dbufs, state, d1, l2_eps=1e-6)

    torch.cuda.synchronize()
    saved = state.clone()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    state.copy_(saved)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    kr = rope_ref(k, pos, sections, True, 1.0e7, rotary).half()
    qrr = rope_ref(q, pos, sections, True, 1.0e7, rotary).half()
    for t in range(prompt, total):
        for b, x in zip(bufs + dbufs, (q, k, v) + dargs):
            b.copy_(x[t:t + 1])
        p1.copy_(pos[:, t:t + 1])
        i1.fill_(t)
        length.fill_(t + 1)
        graph.replay()
        torch.cuda.synchronize()
        # the cached keys are within one rounding of the reference's, and so is the query: half an ulp
        # of each operand moves a score by at most 2 * 2^-11 sum|q k|
        i = torch.arange(t + 1, device="cuda")
        p = table[0].long()[i // page]
        assert (cache.k[p, :, i % page].double() - kr[:t + 1].double()).abs().max() <= 2 ** -10 * 8
        assert (qr.double() - qrr[t:t + 1].double()).abs().max() <= 2 ** -10 * 8
        attention_check(torch, qr, [(cache.k[p, :, i % page], v[:t + 1])], dim ** -0.5, att, lse, f"token {t}")
        ref, s, size = delta_ref(torch, *[x[:t + 1] for x in dargs], torch.zeros(4, 128, 128, device="cuda"), 128 ** -0.5,
                                 1e-6)
        close16(d1[0], ref[t], 2 * (t + 2) * 136 * 2.0 ** -24 * size * 128 ** -0.5, f"delta token {t}")
        if t == prompt:
            close16(dout, ref[:prompt], 2 * (t + 2) * 136 * 2.0 ** -24 * size * 128 ** -0.5, "delta prompt")
