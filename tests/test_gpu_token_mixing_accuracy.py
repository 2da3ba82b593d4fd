"""What the token-mixing operators keep of small terms beside large ones: the
tail of a softmax under one dominant key, the fp32 states of prompts.

Attention's bounds are those of test_gpu_token_mixing, with weights kept to 22
bits or to 2^-40 of the largest one's size.  An output is one rounding to fp16
away from fp32's, so what single outputs cannot show is looked for in their
mean: roundings to nearest are independent of each other and off by at most half
a step, 2^-11 of the value, 2^-11 / sqrt(3) in root mean square, so the mean
relative error of N outputs stays within six times 2^-11 / sqrt(3 N).

A prompt's final states are compared with the recurrence in fp64; they may be
off by eight times what the plain recurrence in fp32 is off by on the same
inputs (chunks round other terms in another order: half to twice of it is
expected, one fp16 operand without its low part makes it a thousand times),
and by the absolute error that the header allows.
"""
import math

import pytest

from test_gpu_token_mixing import attention_setup, close16, delta_inputs, gen, randn

pytestmark = pytest.mark.gpu


def weights_check(torch, q, keys, scale, out, lse, what):
    """Every row against fp64; the mean relative error of the outputs."""
    group = q.shape[1] // keys[0][0].shape[1]
    errors = []
    for b, (k, v) in enumerate(keys):
        if k.shape[0] == 0:
            assert not out[b].any() and (lse[b] == -math.inf).all(), what
            continue
        kk, vv = (x.double().repeat_interleave(group, dim=1).transpose(0, 1) for x in (k, v))
        s = torch.einsum("hd,hnd->hn", q[b].double(), kk) * scale
        # fp32 scores: D products and their scaling
        e = torch.einsum("hd,hnd->hn", q[b].double().abs(), kk.abs()).amax(1) * scale * q.shape[2] * 2.0 ** -24
        p = torch.softmax(s, 1)
        ref, spread = torch.einsum("hn,hnd->hd", p, vv), torch.einsum("hn,hnd->hd", p, vv.abs())
        kept = 2.0 ** -22 * spread + 2.0 ** -40 * p.amax(1)[:, None] * vv.abs().sum(1)
        close16(out[b], ref, spread * (2 * e[:, None] + 2.0 ** -18) + kept, f"{what} row {b}")
        ref_lse = torch.logsumexp(s, 1)
        assert ((lse[b].double() - ref_lse).abs() <= 2 * e + 2.0 ** -20 * (1 + ref_lse.abs())).all(), what
        errors.append(((out[b].double() - ref) / ref).flatten())
    errors = torch.cat(errors)
    return errors.mean().abs().item(), errors.numel()


# ---- attention: one dominant key over a long tail ---------------------------------

@pytest.mark.parametrize("nats", [10.0, 14.0, 18.0, 24.0])
@pytest.mark.parametrize("dim,hq,hk,page,lens,sinks", [
    (128, 8, 8, 16, [4096], 1), (64, 8, 2, 16, [16384, 300], 4), (256, 16, 1, 48, [4096, 0, 1, 5000], 1),
    (128, 32, 8, 16, [1200] * 40, 4)])
def test_attention_sink(cuda, nats, dim, hq, hk, page, lens, sinks):
    """The first keys of a trained model's sequence take most of the weight and have values near 0: what
    the output is made of are the many small weights behind them."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(int(nats) + dim + len(lens))
    q, ck, cv, table, lengths, keys = attention_setup(torch, g, lens, hq, hk, dim, page, qscale=0.3)
    # dimension 0 of q is 1 and that of the dominant keys sqrt(dim) * nats (both exact in fp16 to a part in 2^11, and taken
    # as they are by the reference), of the others 0; tail values of a mean other than 0, so that sums do not cancel
    q[:, :, 0] = 1.0
    for b, n in enumerate(lens):
        if n == 0:
            continue
        k, v = keys[b]
        k[:, :, 0] = 0.0
        v += 2.0
        for i in range(0, min(n, 16 * sinks), 16):
            k[i, :, 0] = math.sqrt(dim) * nats
            v[i] = 0.0
        v *= 1000.0
        i = torch.arange(n, device="cuda")
        p = table[b].long()[i // page]
        ck[p, :, i % page], cv[p, :, i % page] = k, v
    out, lse = torch.empty_like(q), torch.empty(len(lens), hq, device="cuda")
    ws = mcv.paged_attention_workspace(len(lens), hq, hk, dim)
    mcv.paged_attention_decode(q, mcv.PagedKVCache(ck, cv), table, lengths, out, ws, lse=lse)
    weights_check(torch, q, keys, dim ** -0.5, out, lse, f"sink {nats}")


@pytest.mark.parametrize("exponent", [-1, -9, -20])
def test_attention_weights_keep_their_low_bits(cuda, exponent):
    """One key of every 16 dominates and has the value 0; all others weigh 2^exponent (1 + 2^-11) of it each, where a
    single fp16 is off by half a step and always the same way: the outputs' mean error shows what the weights lost."""
    import mcv_b200 as mcv
    torch = cuda
    g = gen(9)
    n, heads, dim = 2001, 16, 128
    q, ck, cv, table, lengths, keys = attention_setup(torch, g, [n], heads, heads, dim, 16)
    q.zero_()
    q[:, :, 0] = 8.0
    k, v = keys[0]
    k.zero_()
    k[::16, :, 0] = 8.0
    # values of one sign, so large that the outputs are normal fp16 numbers
    v.copy_((v.abs() + 1.0) * 4000.0)
    v[::16] = 0.0
    i = torch.arange(n, device="cuda")
    p = table[0].long()[i // 16]
    ck[p, :, i % 16], cv[p, :, i % 16] = k, v
    scale = float(torch.tensor(-math.log(2.0 ** exponent * (1 + 0.99 * 2.0 ** -11)) / 64.0, dtype=torch.float32))
    out, lse = torch.empty_like(q), torch.empty(1, heads, device="cuda")
    mcv.paged_attention_decode(q, mcv.PagedKVCache(ck, cv), table, lengths, out,
                               mcv.paged_attention_workspace(1, heads, heads, dim), scale=scale, lse=lse)
    mean, count = weights_check(torch, q, keys, scale, out, lse, "equal weights")
    # the score, 2^exponent's logarithm, is a product and a sum in fp32: up to 20 (2^-24 + 2^-24) of the weights more
    assert mean <= 6 * 2.0 ** -11 / math.sqrt(3 * count) + 2.0 ** -18, mean


@pytest.mark.parametrize("n", [1, 37, 3000])
def test_attention_small_lse(cuda, n):
    """Sums near 1: the log-sum-exp is as small as the weights behind the largest, and keeps fp32's accuracy for it."""
    import mcv_b200 as mcv
    torch = cuda
    q, ck, cv, table, lengths, keys = attention_setup(torch, gen(n), [n], 2, 2, 64, 16)
    q.zero_()
    q[:, :, 0] = 1.0
    i = torch.arange(n, device="cuda")
    ck[table[0].long()[i // 16], :, i % 16] = 0.0
    ck[table[0].long()[i[1:] // 16], :, i[1:] % 16, 0] = -16.0
    out, lse = torch.empty_like(q), torch.empty(1, 2, device="cuda")
    mcv.paged_attention_decode(q, mcv.PagedKVCache(ck, cv), table, lengths, out, mcv.paged_attention_workspace(1, 2, 2, 64),
                               scale=1.0, lse=lse)
    ref = math.log1p((n - 1) * math.exp(-16.0))
    # Each addition to a sum near 1 rounds by at most 2^-24, half a step there; the terms are equal, so roundings may all
    # go one way.  A sum with the largest weight in it meets one addition per unit of 16 keys of its warp, three across
    # lanes, three across warps and one per further block (of four units or more): no more than n / 16 + 6.  The
    # logarithm adds a few 2^-24 of its value.
    assert ((lse.double() - ref).abs() <= (n / 16 + 8) * 2.0 ** -24).all(), (lse, ref)


# ---- the gated delta rule: states of prompts -------------------------------------------

def recurrence(torch, q, k, v, g, beta, s, dtype):
    """Token by token, in this type, with q and k normalised."""
    r = v.shape[1] // q.shape[1]

    def prep(x):
        x = x.to(dtype)
        return (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(r, dim=1)

    q, k, v, beta = prep(q), prep(k), v.to(dtype), beta.to(dtype)
    decay = torch.exp(g.to(dtype))
    s = s.to(dtype).clone()
    out = torch.empty_like(v)
    for t in range(v.shape[0]):
        s = s * decay[t][:, None, None]
        u = beta[t][:, None] * (v[t] - (s * k[t][:, :, None]).sum(1))
        s = s + k[t][:, :, None] * u[:, None]
        out[t] = (s * q[t][:, :, None]).sum(1)
    return out, s


def prompt(torch, g, kind, n, hk, hv, dk, dv):
    q, k, v, gl, beta = delta_inputs(torch, g, n, hk, hv, dk, dv)
    v = v.clone()
    start = randn(g, 1, hv, dk, dv, dtype=torch.float32)
    if kind.startswith("reset"):          # one large value, small ones behind it, and a decay between them
        v *= 0.01
        v[0] = 30000.0
        start.zero_()
        gl[8] = -float(kind[5:])
    elif kind == "forget":
        gl[::7] = -300.0
        gl[50] = -math.inf
    elif kind == "keep":
        gl.zero_()
    elif kind == "write":
        beta.fill_(1.0)
        gl.zero_()
        k = k[:1].expand(n, hk, dk).contiguous()
    elif kind == "mixed":
        gl = gl * torch.randint(0, 2, gl.shape, generator=g, device="cuda") * 40
    elif kind == "steps":                 # values of another size every 50 tokens, long-lived states
        e = torch.randint(-7, 8, (n // 50 + 1,), generator=g, device="cuda").repeat_interleave(50)[:n]
        v *= (2.0 ** e.float()).half()[:, None, None]
        gl *= 0.1
    return q, k, v, gl, beta, start


@pytest.mark.parametrize("heads", [2, 20, 40])     # one and two column groups a block, whole heads
@pytest.mark.parametrize("kind,n", [("plain", 64), ("plain", 700), ("reset40", 64), ("reset40", 200), ("reset14", 64),
                                    ("reset14", 200), ("forget", 200), ("keep", 200), ("write", 200), ("mixed", 200),
                                    ("steps", 900)])
@pytest.mark.parametrize("dk", [64, 128])
def test_prefill_states(cuda, heads, kind, n, dk):
    import mcv_b200 as mcv
    torch = cuda
    g = gen(n + heads + dk)
    hk = heads // 2 if kind == "plain" else heads
    q, k, v, gl, beta, start = prompt(torch, g, kind, n, hk, heads, dk, 128)
    out, new = torch.empty(n, heads, 128, dtype=torch.float16, device="cuda"), torch.empty_like(start)
    ws = mcv.gated_delta_workspace(n, 1, heads, dk, 128)
    mcv.device_errors()
    mcv.gated_delta_prefill(q, k, v, gl, beta, torch.tensor([0, n], dtype=torch.int32, device="cuda"), start, out, ws,
                            state_out=new, scale=1.0, l2_eps=1e-6)
    assert mcv.device_errors() == 0
    ref_out, ref = recurrence(torch, q, k, v, gl, beta, start[0], torch.float64)
    fp32_out, fp32 = recurrence(torch, q, k, v, gl, beta, start[0], torch.float32)
    # 2^-36, where whole heads are taken of the largest value or state
    large = max(1.0, v.abs().max().item(), start.abs().max().item()) if heads == 40 else 1.0
    least = 2.0 ** -36 * large
    err, plain = (new[0].double() - ref).abs().max().item(), (fp32.double() - ref).abs().max().item()
    assert err <= 8 * plain + least, f"states off by {err:.3g}, fp32's by {plain:.3g}, absolute {least:.3g}"
    # an output's error is that of a state's column times q of norm 1, and its rounding
    wrong = (out.double() - ref_out).abs() - 2.0 ** -11 * ref_out.abs() - 2.0 ** -25
    off = (fp32_out.double() - ref_out).abs()
    for rows in (slice(0, 9), slice(9, None)):
        err, plain = wrong[rows].max().item(), off[rows].max().item()
        assert err <= 8 * plain + math.sqrt(dk) * least, f"outputs off by {err:.3g}, fp32's by {plain:.3g}"
