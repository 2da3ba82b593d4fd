"""Calls at the edges of the token-mixing operators: the largest write
strength, two calls at once, graphs that share a workspace, gaps between
sequences, the largest batch, and the same numbers whatever the split.

Where results are compared with 64-bit ones the tolerances are those of
test_gpu_token_mixing; a write strength of up to 2 doubles what a token's
rounding errors add to the state, so its bound is doubled.
"""
import pytest

from test_gpu_token_mixing import close16, delta_check, delta_inputs, delta_ref, gen, randn

pytestmark = pytest.mark.gpu


def cu_of(torch, *bounds):
    return torch.tensor(bounds, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("heads", [2, 20, 40])     # one and two column groups a block, whole heads
@pytest.mark.parametrize("same_key", [True, False])
def test_prefill_largest_write_strength(cuda, heads, same_key):
    """beta = 2 reflects the state along each key: with one key again and again the triangular inverse has
    entries of 4, its largest."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(5)
    n, dk = 150, 128
    q, k, v, gl, beta = delta_inputs(torch, g, n, heads, heads, dk, 128)
    beta.fill_(2.0)
    if same_key:
        k = k[:1].expand(n, heads, dk).contiguous()
        gl.zero_()
    state = randn(g, 1, heads, dk, 128, dtype=torch.float32)
    out, new = torch.empty(n, heads, 128, dtype=torch.float16, device="cuda"), torch.empty_like(state)
    mcv.gated_delta_prefill(q, k, v, gl, beta, cu_of(torch, 0, n), state, out,
                            mcv.gated_delta_workspace(n, 1, heads, dk, 128), state_out=new, l2_eps=1e-6)
    ref, s, size = delta_ref(torch, q, k, v, gl, beta, state[0], dk ** -0.5, 1e-6)
    fp32 = 2 * (n + 1) * (dk + 8) * 2.0 ** -24 * size
    close16(out, ref, 2 * fp32[None] * dk ** -0.5, "out")
    assert ((new[0].double() - s).abs() <= fp32[:, None] + 2.0 ** -24 * s.abs()).all()


def test_prefill_gaps_and_empty_sequences(cuda):
    """Rows before the first and behind the last sequence stay; empty sequences pass their states on."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(6)
    bounds = [5, 5, 5, 70, 70, 71, 199, 199]
    args = delta_inputs(torch, g, 210, 2, 4, 64, 48)
    state = randn(g, 7, 4, 64, 48, dtype=torch.float32)
    out = torch.full((210, 4, 48), 3.0, dtype=torch.float16, device="cuda")
    new = torch.full_like(state, 9.0)
    mcv.gated_delta_prefill(*args, cu_of(torch, *bounds), state, out, mcv.gated_delta_workspace(210, 7, 4, 64, 48),
                            state_out=new, l2_eps=1e-6)
    assert (out[:5] == 3.0).all() and (out[199:] == 3.0).all()
    for i, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
        if lo == hi:
            assert torch.equal(new[i], state[i])
        else:
            delta_check(torch, [x[lo:hi] for x in args], state[i], out[lo:hi], new[i], 64 ** -0.5, 1e-6, f"sequence {i}")


def test_step_largest_batch(cuda):
    import mcv_b200 as mcv
    torch = cuda
    g = gen(7)
    n = 65535
    args = delta_inputs(torch, g, n, 1, 1, 64, 16)
    state = randn(g, n, 1, 64, 16, dtype=torch.float32)
    out, new = torch.empty(n, 1, 16, dtype=torch.float16, device="cuda"), torch.empty_like(state)
    mcv.gated_delta_step(*args, state, out, state_out=new, l2_eps=1e-6)
    for b in (0, 1, 32768, n - 1):
        delta_check(torch, [x[b:b + 1] for x in args], state[b], out[b:b + 1], new[b], 0.125, 1e-6, f"sequence {b}")
    with pytest.raises(RuntimeError):
        wide = [torch.cat([x, x[:1]]) for x in args]
        mcv.gated_delta_step(*wide, torch.cat([state, state[:1]]), torch.empty(n + 1, 1, 16, dtype=torch.float16,
                                                                               device="cuda"))


def attention_case(torch, mcv, seed, batch, longest, hq, hk, dim, page):
    g = gen(seed)
    cols = -(-longest // page)
    cache = mcv.PagedKVCache(randn(g, batch * cols, hk, page, dim), randn(g, batch * cols, hk, page, dim))
    table = torch.randperm(batch * cols, generator=g, device="cuda").int().view(batch, cols)
    lengths = torch.randint(0, longest + 1, (batch,), generator=g, device="cuda").int()
    lengths[0] = longest
    return [randn(g, batch, hq, dim), cache, table, lengths, torch.empty(batch, hq, dim, dtype=torch.float16, device="cuda")]


def test_two_streams_at_once(cuda):
    """Attention and prompts on two streams, each with a workspace of its own, give what they give alone."""
    import mcv_b200 as mcv
    torch = cuda
    att = [attention_case(torch, mcv, i, 3, 5000, 16, 2, 128, 16) for i in (1, 2)]
    wss = [mcv.paged_attention_workspace(3, 16, 2, 128) for _ in att]
    n, heads = 500, 40
    deltas = [delta_inputs(torch, gen(10 + i), n, heads, heads, 128, 128) for i in range(2)]
    wsd = [mcv.gated_delta_workspace(n, 1, heads, 128, 128) for _ in deltas]
    outs = [torch.empty(n, heads, 128, dtype=torch.float16, device="cuda") for _ in deltas]
    states = [torch.empty(1, heads, 128, 128, device="cuda") for _ in deltas]
    cu = cu_of(torch, 0, n)

    def run(i, stream=None):
        mcv.paged_attention_decode(*att[i], wss[i], stream=stream)
        mcv.gated_delta_prefill(*deltas[i], cu, None, outs[i], wsd[i], state_out=states[i], l2_eps=1e-6, stream=stream)

    alone = []
    for i in range(2):
        run(i)
        torch.cuda.synchronize()
        alone.append([x.clone() for x in (att[i][-1], outs[i], states[i])])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for x in (*(a[-1] for a in att), *outs, *states):
        x.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            run(i, streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(alone[i], (att[i][-1], outs[i], states[i])):
            assert torch.equal(a, b)


def test_graphs_share_a_workspace(cuda):
    """Two captured calls of different shapes on one workspace, replayed in turn on one stream, with an eager call
    between them."""
    import mcv_b200 as mcv
    torch = cuda
    cases = [attention_case(torch, mcv, 21, 1, 30000, 16, 2, 256, 16), attention_case(torch, mcv, 22, 37, 700, 8, 2, 256, 64),
             attention_case(torch, mcv, 23, 2, 9, 8, 2, 256, 3)]
    ws = mcv.paged_attention_workspace(64, 16, 2, 256)
    want = []
    for c in cases:
        mcv.paged_attention_decode(*c, mcv.paged_attention_workspace(64, 16, 2, 256))
        want.append(c[-1].clone())
    side = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for c in cases[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            mcv.paged_attention_decode(*c, ws)
            mcv.paged_attention_decode(*c, ws)
        graphs.append(graph)
    for c in cases:
        c[-1].zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(5):
            graphs[0].replay()
            mcv.paged_attention_decode(*cases[2], ws)
            graphs[1].replay()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c[-1], w)


@pytest.mark.parametrize("dim,rotary,hq,hk", [(64, 32, 12, 3), (128, 128, 8, 8), (256, 64, 8, 2), (256, 256, 40, 4),
                                              (80, 32, 5, 1)])
def test_mrope_however_many_tokens(cuda, dim, rotary, hq, hk):
    """A long call, whose tokens have a warp each, and short ones, whose warps share them, agree bit for bit; so
    does rotating in place."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(dim + rotary)
    n, page = 3001, 16
    q, k, v = randn(g, n, hq, dim), randn(g, n, hk, dim), randn(g, n, hk, dim)
    rope = mcv.MRope(rotary, [rotary // 2 - 2 * (rotary // 6), rotary // 6, rotary // 6], True)
    pos = torch.randint(0, 100000, (3, n), generator=g, device="cuda").int()
    cols = -(-n // page)
    table = torch.randperm(cols, generator=g, device="cuda").int()[None].contiguous()
    idx = torch.arange(n, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(idx)
    got = []
    for piece in (n, 613, 40, 1):
        cache = mcv.PagedKVCache.empty(cols, hk, page, dim)
        cache.k.zero_()
        cache.v.zero_()
        qo = torch.zeros_like(q)
        for at in range(0, n if piece > 1 else 5, piece):
            s = slice(at, min(at + piece, n))
            mcv.mrope_append_kv(q[s], k[s], v[s], pos[:, s].contiguous(), rope, cache, table, idx[s], qo[s], seq=seq[s])
        got.append((qo, cache.k, cache.v))
    for qo, ck, cv in got[1:3]:
        assert torch.equal(qo, got[0][0]) and torch.equal(ck, got[0][1]) and torch.equal(cv, got[0][2])
    assert torch.equal(got[3][0][:5], got[0][0][:5])
    mcv.mrope(q, pos, rope, q)
    assert torch.equal(q, got[0][0])


@pytest.mark.parametrize("page,hq,hk,dim", [(1, 8, 2, 64), (1000, 16, 2, 256), (5000, 5, 1, 128), (3, 34, 2, 64)])
def test_pages_of_any_size(cuda, page, hq, hk, dim):
    """A cache written token by token through its pages reads like one piece: pages of one key, pages longer than the
    sequences, 17 query heads a kv head."""
    import mcv_b200 as mcv
    from test_gpu_token_mixing import attention_check
    torch = cuda
    g = gen(page + hq)
    lens = [1, 40, 333]
    cols = -(-333 // page)
    total = sum(lens)
    cache = mcv.PagedKVCache.empty(3 * cols, hk, page, dim)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    table = torch.randperm(3 * cols, generator=g, device="cuda").int().view(3, cols)
    q, k, v = randn(g, total, hq, dim), randn(g, total, hk, dim), randn(g, total, hk, dim)
    rope = mcv.MRope(32, [16])
    index = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).int().cuda()
    still = torch.zeros(1, total, dtype=torch.int32, device="cuda")       # position 0: keys stay as they are
    mcv.mrope_append_kv(q, k, v, still, rope, cache, table, index, torch.empty_like(q), seq=seq)
    qs = randn(g, 3, hq, dim)
    out, lse = torch.empty(3, hq, dim, dtype=torch.float16, device="cuda"), torch.empty(3, hq, device="cuda")
    mcv.paged_attention_decode(qs, cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out,
                               mcv.paged_attention_workspace(3, hq, hk, dim), lse=lse)
    keys, at = [], 0
    for n in lens:
        keys.append((k[at:at + n], v[at:at + n]))
        at += n
    attention_check(torch, qs, keys, dim ** -0.5, out, lse, "pages")
    assert mcv.device_errors() == 0


def test_mrope_turns_back(cuda):
    """Negative positions turn the other way: there and back leaves two roundings, each half a step of a vector of the
    pair's length, and what fp32 leaves of two rotations (2^-19 of it)."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(31)
    x = randn(g, 77, 4, 128)
    pos = torch.randint(0, 200000, (1, 77), generator=g, device="cuda").int()
    rope = mcv.MRope(128, [64])
    there, back = torch.empty_like(x), torch.empty_like(x)
    mcv.mrope(x, pos, rope, there)
    mcv.mrope(there, -pos, rope, back)
    length = (x[..., :64].double() ** 2 + x[..., 64:].double() ** 2).sqrt().repeat(1, 1, 2)
    # the first rounding errs by 2^-11 in each of a pair's two, turned: sqrt 2 times that at most
    assert ((back.double() - x.double()).abs() <= (2.0 ** -11 * (1 + 2.0 ** 0.5) + 2.0 ** -19) * length + 2.0 ** -23).all()


@pytest.mark.parametrize("dim,tokens,gap", [(64, 700, 8), (128, 33, 24), (256, 4000, 8)])
def test_mrope_in_place_again_and_again(cuda, dim, tokens, gap):
    """In place, with rows that share 32-byte sectors, each call's input written by the call before it, without a wait
    between them: the same bits as call by call into fresh tensors."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(dim)
    heads, rope = 9, mcv.MRope(dim, [dim // 2 - 8, 4, 4], interleaved=False)
    pos = torch.randint(0, 5000, (3, tokens), generator=g, device="cuda", dtype=torch.int32)
    x = torch.zeros(tokens, heads, dim + gap, dtype=torch.float16, device="cuda")[:, :, :dim]
    x.copy_(randn(g, tokens, heads, dim))
    step = x.contiguous()
    for _ in range(6):
        out = torch.empty_like(step)
        mcv.mrope(step, pos, rope, out)
        torch.cuda.synchronize()
        step = out
    for _ in range(6):
        mcv.mrope(x, pos, rope, x)
    assert torch.equal(x, step)


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("heads", [2, 20, 40])     # one and two column groups a block, whole heads
@pytest.mark.parametrize("kind", ["start", "sum", "within"])
def test_prefill_beyond_its_range(cuda, heads, dk, kind):
    """States and sums of values beyond the documented range: either the result is right or the call is reported; the
    largest within it are right and not reported."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(heads)
    n = 130
    q, k, v, gl, beta = delta_inputs(torch, g, n, heads, heads, dk, 128)
    v = v.clone()
    k = k[:1].expand(n, heads, dk).contiguous()
    gl.zero_()
    beta.fill_(1.0)
    state = torch.zeros(1, heads, dk, 128, device="cuda")
    if kind == "start":
        state[0, 0, 3, 5] = 1.0e6
    elif kind == "sum":           # opposite keys of one direction: u takes twice the value again and again
        k[1::2] *= -1
        v[:, 0, 7] = 60000.0
    else:
        v[0, 0, 7] = 60000.0
    out, new = torch.empty(n, heads, 128, dtype=torch.float16, device="cuda"), torch.empty_like(state)
    ws = mcv.gated_delta_workspace(n, 1, heads, dk, 128)
    mcv.device_errors()
    mcv.gated_delta_prefill(q, k, v, gl, beta, cu_of(torch, 0, n), state, out, ws, state_out=new, scale=2.0 ** -10,
                            l2_eps=1e-6)
    errors = mcv.device_errors()
    assert errors == (0 if torch.isfinite(new).all() else 4)
    if kind == "within":
        assert errors == 0
    elif kind == "start" and heads < 40:
        assert errors == 4
    if errors == 0:
        ref, s, size = delta_ref(torch, q, k, v, gl, beta, state[0], 2.0 ** -10, 1e-6)
        fp32 = (n + 1) * (dk + 8) * 2.0 ** -24 * size
        assert ((new[0].double() - s).abs() <= fp32[:, None] + 2.0 ** -24 * s.abs()).all()
    if kind != "start":           # reported without final states too
        mcv.gated_delta_prefill(q, k, v, gl, beta, cu_of(torch, 0, n), None, out, ws, scale=2.0 ** -10, l2_eps=1e-6)
        assert mcv.device_errors() == errors


@pytest.mark.parametrize("pages,heads,page", [(9, 1, 16), (9, 2, 1), (1, 1, 128), (1, 2, 128)])
def test_caches_and_rows_of_size_one(cuda, pages, heads, page):
    """Dimensions of size 1 with strides of their own - one kv head, pages of one slot, one page, one token of a row whose
    width is no multiple of 8 - give what the dense tensors give; other layouts are refused."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(page)
    n, dim = min(pages * page, 100), 64
    dense = mcv.PagedKVCache(randn(g, pages, heads, page, dim), randn(g, pages, heads, page, dim))
    shape, stride = (pages, heads, page, dim), list(dense.k.stride())
    for i in range(3):
        if shape[i] == 1:
            stride[i] = 8 * (i + 1) + 1
    odd = mcv.PagedKVCache(*(x.clone().as_strided(shape, stride) for x in (dense.k, dense.v)))
    table = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    wide = randn(g, 1, 3 * 4 * dim + 1)
    assert wide[:, :dim].stride(0) % 8
    q = wide[:, :4 * dim].view(1, 4, dim)
    k, v = (wide[:, at * 4 * dim:][:, :heads * dim].view(1, heads, dim) for at in (1, 2))
    rope, pos = mcv.MRope(dim, [dim // 2]), torch.tensor([[5]], dtype=torch.int32, device="cuda")
    index, lengths = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (n - 1, n))
    ws, got = mcv.paged_attention_workspace(1, 4, heads, dim), []
    for cache, rows in ((dense, [x.contiguous() for x in (q, k, v)]), (odd, [q, k, v])):
        turned, out = torch.empty(1, 4, dim, dtype=torch.float16, device="cuda"), torch.empty_like(q).contiguous()
        mcv.mrope_append_kv(*rows, pos, rope, cache, table, index, turned)
        mcv.paged_attention_decode(turned, cache, table, lengths, out, ws)
        got.append((turned, out, cache.k.clone(), cache.v.clone()))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    for bad in (torch.empty(4, 2, dim, 16, dtype=torch.float16, device="cuda").transpose(2, 3),
                torch.empty(4, 16, 2, dim, dtype=torch.float16, device="cuda").transpose(1, 2)):
        with pytest.raises(RuntimeError, match="contiguous"):
            mcv.PagedKVCache(bad, bad)
        with pytest.raises(RuntimeError, match="laid out alike"):
            mcv.PagedKVCache(bad.contiguous(), bad)


@pytest.mark.parametrize("dk,dv,batch,heads", [(64, 16, 10, 20), (128, 16, 10, 40), (128, 32, 10, 20), (64, 32, 10, 14),
                                               (128, 48, 5, 20), (64, 80, 3, 60)])
def test_prefill_narrow_values(cuda, dk, dv, batch, heads):
    """More heads than SMs with few value columns each."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(dv + heads)
    n = 70
    q, k, v, gl, beta = delta_inputs(torch, g, batch * n, heads, heads, dk, dv)
    state = randn(g, batch, heads, dk, dv, dtype=torch.float32)
    out, new = torch.empty(batch * n, heads, dv, dtype=torch.float16, device="cuda"), torch.empty_like(state)
    mcv.gated_delta_prefill(q, k, v, gl, beta, cu_of(torch, *range(0, batch * n + 1, n)), state, out,
                            mcv.gated_delta_workspace(batch * n, batch, heads, dk, dv), state_out=new, l2_eps=1e-6)
    for b in (0, batch // 2, batch - 1):
        rows = slice(b * n, (b + 1) * n)
        delta_check(torch, [x[rows] for x in (q, k, v, gl, beta)], state[b], out[rows], new[b], dk ** -0.5, 1e-6, f"sequence {b}")
