"""Attention with a relative position bias and the per-head norm with rotation, against 64-bit definitions.

Bounds are elementwise and counted: u = finfo(dtype).eps / 2 is the relative error of one rounding, `tiny` half a step of
the dtype's smallest values.  What is rounded: the operands p and ds of the products, the stored outputs, and the output that
delta = rowsum(dout * out) is formed from.  fp32 arithmetic on scores of a few tens leaves less than F32 of a sum of terms."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
F32 = 3e-5


def ops():
    from pytorch_distributed_training_amd import ops as o

    return o


def half_step(dtype):
    return torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def bucket_rule(gap, buckets, max_distance):
    half = buckets // 2
    exact, m = half // 2, half - half // 2

    def one(n):
        if n < exact:
            return n
        return exact + max(j for j in range(m) if n ** m * exact ** j >= max_distance ** j * exact ** m)

    side = torch.tensor([one(n) for n in range(int(gap.abs().max()) + 1)], device=gap.device)
    return side[gap.abs()] + half * (gap > 0)


def keep_mask(rng, p, site, B, A, S):
    """The dropout decisions of (sample, head, query, key), written out in whole numbers."""
    M = 0xFFFFFFFF

    def mix(x):
        for shift, mul in ((16, 0x7FEB352D), (15, 0x846CA68B)):
            x = ((x ^ (x >> shift)) * mul) & M
        return x ^ (x >> 16)

    seed, off = (int(t) for t in rng.state.tolist())
    mixed = (seed ^ ((off * 0x9E3779B97F4A7C15) & (2 ** 64 - 1))) & (2 ** 64 - 1)
    ids = rng.sample_ids.long() if rng.sample_ids is not None else torch.arange(B, device="cuda")
    bh = ((ids[:, None] * A + torch.arange(A, device="cuda")) & M)[:, :, None]
    q = torch.arange(S, device="cuda")
    row = mix((q ^ (mixed & M)) & M)[None, None, :]
    row = mix((row ^ ((bh * 0x9E3779B9) & M) ^ (mixed >> 32) ^ ((site * 0x85EBCA6B) & M) ^ ((rng.counter * 0xC2B2AE35) & M)) & M)
    x = (row[..., None] ^ ((q * 0x9E3779B9) & M)) & 0xFFFFFF
    return ((x * 0xEBCA6B) & M) >= (round(p * 65536) << 16)


def check_attention(q, k, v, bias, dout, *, max_distance=128, valid=None, spans=None, keep=None, p_drop=0.0, got, table_dtype=None):
    """`got` = (out, dq, dk, dv, dbias) against the formulas in 64 bits, sample by sample."""
    dtype = q.dtype
    u, tiny = half_step(dtype)
    A, D = q.shape[-2:]
    scale = 1 / math.sqrt(D)
    flat = [t.detach().reshape(-1, A, D) for t in (q, k, v, dout)]
    outs = [t.reshape(-1, A, D).double() if t is not None else None for t in got[:4]]
    db = torch.zeros(bias.shape if bias is not None else (1, A), dtype=torch.float64, device="cuda")
    db_tol = torch.zeros_like(db)

    def close(x, ref, tol, what):
        bad = ((x - ref).abs() > tol) | ~torch.isfinite(x)
        assert not bad.any(), (what, int(bad.sum()), float((x - ref).abs().max()), float(((x - ref).abs() / tol.clamp(min=1e-300)).max()))

    for b, (lo, hi) in enumerate(spans):
        n = hi - lo
        if n == 0:
            continue
        ok = valid[b] if valid is not None else torch.ones(n, dtype=torch.bool, device="cuda")
        qq, kk, vv, gg = (t[lo:hi].transpose(0, 1).double() for t in flat)
        kk, vv = (torch.where(ok[None, :, None], t, 0.0) for t in (kk, vv))
        s = qq @ kk.transpose(1, 2) * scale
        place = torch.arange(n, device="cuda")
        if bias is not None:
            bucket = bucket_rule(place[None, :] - place[:, None], bias.shape[0], max_distance)
            s = s + bias.detach().double()[bucket].permute(2, 0, 1)
        s = s.masked_fill(~ok, -math.inf)
        P = torch.softmax(s, -1) if ok.any() else torch.zeros_like(s)
        Z = (keep[b].double() / (1 - p_drop)) if keep is not None else torch.ones_like(P)
        O = (P * Z) @ vv
        f = u + F32
        # a probability below the smallest normal value loses up to `tiny` of the row's largest
        lost = tiny * ok.sum() * Z.amax() * vv.abs().amax()
        O_tol = f * ((P * Z) @ vv.abs() + O.abs()) + lost + tiny
        close(outs[0][lo:hi].transpose(0, 1), O, O_tol, "out")
        if got[1] is None:
            continue
        dP = gg @ vv.transpose(1, 2) * Z
        ds = P * (dP - (P * dP).sum(-1, keepdim=True))
        # ds carries the error of delta, which is formed from the rounded output, and its own rounding as an operand
        d_delta = (gg.abs() * (u * O.abs() + u * ((P * Z) @ vv.abs()) + lost + tiny)).sum(-1, keepdim=True) + F32 * (gg.abs() * O.abs()).sum(-1, keepdim=True)
        e = P * d_delta + F32 * P * ((gg.abs() @ vv.abs().transpose(1, 2)) * Z + dP.abs())
        e_op = e + u * ds.abs() + tiny
        P_op = f * P * Z + tiny * Z
        dq, dk, dv = ds @ kk * scale, ds.transpose(1, 2) @ qq * scale, (P * Z).transpose(1, 2) @ gg
        close(outs[1][lo:hi].transpose(0, 1), dq, scale * (e_op @ kk.abs()) + f * dq.abs() + tiny, "dq")
        # (operands of keys that nothing attends to are exact zeros)
        live = ok[None, :, None].double()
        close(outs[2][lo:hi].transpose(0, 1), dk, live * (scale * (e_op.transpose(1, 2) @ qq.abs()) + f * dk.abs() + tiny), "dk")
        close(outs[3][lo:hi].transpose(0, 1), dv, live * (P_op.transpose(1, 2) @ gg.abs() + f * dv.abs() + tiny), "dv")
        if bias is not None:
            flatb = bucket.flatten()
            db.index_add_(0, flatb, ds.flatten(1).t().contiguous())
            db_tol.index_add_(0, flatb, (e + F32 * ds.abs()).flatten(1).t().contiguous())
    if bias is not None and got[4] is not None:
        ub = half_step(table_dtype or bias.dtype)[0]
        close(got[4].double(), db, db_tol + (ub + F32) * db.abs() + 1e-30 + half_step(table_dtype or bias.dtype)[1], "dbias")


def padded_case(dtype, B, S, A, D, *, lens=None, holes=False, buckets=32, seed=0, bias_dtype=None, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(B, S, 3, A, D, generator=gen, device="cuda") * scale).to(dtype)
    bias = (torch.randn(buckets, A, generator=gen, device="cuda")).to(bias_dtype or dtype)
    dout = (torch.randn(B, S, A, D, generator=gen, device="cuda") * 0.25).to(dtype)
    valid = None
    if lens is not None:
        valid = torch.arange(S, device="cuda")[None, :] < torch.tensor(lens, device="cuda")[:, None]
        if holes:
            valid &= torch.rand(B, S, generator=gen, device="cuda") < 0.6
    return [qkv[:, :, i].requires_grad_() for i in range(3)], bias.requires_grad_(), dout, valid


def spans_of(B, S):
    return [(b * S, (b + 1) * S) for b in range(B)]


# lengths around the 16-, 32-, 64- and 128-row tiles, one token, and lengths whose far tiles use the constant bias
SHAPES = [(1, 1, 1, 64), (2, 2, 3, 64), (1, 15, 2, 64), (3, 17, 2, 32), (2, 33, 1, 128), (1, 63, 2, 96), (2, 64, 2, 64), (1, 65, 2, 8),
          (2, 100, 2, 72), (2, 128, 2, 64), (1, 129, 2, 64), (1, 192, 1, 128), (1, 257, 2, 64), (1, 511, 1, 40), (1, 700, 1, 64),
          (1, 1023, 1, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,S,A,D", SHAPES)
def test_relative_attention_all_keys(dtype, B, S, A, D):
    (q, k, v), bias, dout, _ = padded_case(dtype, B, S, A, D, seed=S)
    out = ops().relative_attention(q, k, v, bias)
    grads = torch.autograd.grad(out, (q, k, v, bias), dout)
    check_attention(q, k, v, bias, dout, spans=spans_of(B, S), got=(out, *grads))
    with torch.no_grad():  # without a tape: the same numbers
        assert torch.equal(ops().relative_attention(q, k, v, bias), out)


@pytest.mark.parametrize("D,B,S,A", [(64, 40, 300, 12), (128, 20, 300, 12), (64, 18, 130, 16), (32, 3, 1500, 16)])
@pytest.mark.parametrize("packed", [False, True])
def test_relative_attention_large_grids(D, B, S, A, packed):
    """Enough workgroups for the 128-row shape of every kernel; ragged lengths, one sample without keys."""
    lens = [0, S, 1] + [S - 7 * i for i in range(B - 3)]
    dtype = torch.bfloat16
    if packed:
        T = sum(lens)
        gen = torch.Generator(device="cuda").manual_seed(T)
        qkv = torch.randn(T, 3, A, D, generator=gen, device="cuda").to(dtype)
        q, k, v = (qkv[:, i].requires_grad_() for i in range(3))
        bias = torch.randn(32, A, generator=gen, device="cuda").to(dtype).requires_grad_()
        dout = (torch.randn(T, A, D, generator=gen, device="cuda") * 0.25).to(dtype)
        cu = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
        out = ops().relative_attention(q, k, v, bias, cu_seqlens=cu, max_seqlen=S)
        spans, valid = list(zip(cu.tolist()[:-1], cu.tolist()[1:])), None
    else:
        (q, k, v), bias, dout, valid = padded_case(dtype, B, S, A, D, lens=lens)
        out = ops().relative_attention(q, k, v, bias, key_mask=valid)
        spans = spans_of(B, S)
    grads = torch.autograd.grad(out, (q, k, v, bias), dout)
    check_attention(q, k, v, bias, dout, valid=valid, spans=spans, got=(out, *grads))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("holes", [False, True])
@pytest.mark.parametrize("S,lens", [(40, [40, 1, 0, 17]), (128, [0, 128, 64, 65]), (200, [3, 129, 200]), (330, [330, 0, 70])])
def test_relative_attention_key_masks_and_garbage(dtype, holes, S, lens):
    B, A, D = len(lens), 2, 64
    (q, k, v), bias, dout, valid = padded_case(dtype, B, S, A, D, lens=lens, holes=holes, seed=S + holes)
    with torch.no_grad():  # what lies behind a masked key takes no part
        junk = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").to(dtype)[torch.arange(B * S, device="cuda").view(B, S) % 3]
        for t in (k, v):
            t[~valid] = junk[~valid][:, None, None]
    for mask in (valid, valid.to(torch.uint8) * 3, valid.int(), valid.long()):
        out = ops().relative_attention(q, k, v, bias, key_mask=mask)
        grads = torch.autograd.grad(out, (q, k, v, bias), dout)
        if mask is valid:
            check_attention(q, k, v, bias, dout, valid=valid, spans=spans_of(B, S), got=(out, *grads))
            first = (out, *grads)
            assert grads[1][~valid].abs().max() == 0 and grads[2][~valid].abs().max() == 0
            for b in range(B):
                if not valid[b].any():
                    assert out[b].abs().max() == 0 and grads[0][b].abs().max() == 0
        else:
            assert all(torch.equal(a, b) for a, b in zip(first, (out, *grads)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,tail", [([5], 0), ([1, 0, 64, 31], 3), ([128, 127, 0, 129, 1], 0), ([300, 2, 190], 70)])
def test_relative_attention_packed_rows(dtype, D, lens, tail):
    A, T = 2, sum(lens) + tail
    gen = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(T, 3, A, D, generator=gen, device="cuda").to(dtype)
    q, k, v = (qkv[:, i].requires_grad_() for i in range(3))
    bias = torch.randn(32, A, generator=gen, device="cuda").requires_grad_()
    dout = (torch.randn(T, A, D, generator=gen, device="cuda") * 0.25).to(dtype)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
    out = ops().relative_attention(q, k, v, bias, cu_seqlens=cu, max_seqlen=max(lens) + 7)
    grads = torch.autograd.grad(out, (q, k, v, bias), dout)
    spans = list(zip(cu.tolist()[:-1], cu.tolist()[1:]))
    check_attention(q, k, v, bias, dout, spans=spans, got=(out, *grads))
    for t in (out, *grads[:3]):  # rows that belong to no sequence
        assert t[sum(lens):].abs().sum() == 0
    # the same rows, one sequence at a time in the padded form
    for lo, hi in spans:
        if hi > lo:
            one = ops().relative_attention(q[None, lo:hi].detach(), k[None, lo:hi].detach(), v[None, lo:hi].detach(), bias.detach())
            assert torch.equal(one[0], out[lo:hi])


@pytest.mark.parametrize("buckets,max_distance", [(4, 2), (4, 512), (6, 9), (16, 64), (32, 128), (32, 200), (64, 100), (126, 512), (128, 33)])
@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.float16])
def test_relative_attention_tables(buckets, max_distance, bias_dtype):
    S, A = 600, 2
    (q, k, v), bias, dout, _ = padded_case(torch.float16, 1, S, A, 64, buckets=buckets, bias_dtype=bias_dtype, seed=buckets + max_distance)
    out = ops().relative_attention(q, k, v, bias, max_distance=max_distance)
    grads = torch.autograd.grad(out, (q, k, v, bias), dout)
    check_attention(q, k, v, bias, dout, max_distance=max_distance, spans=spans_of(1, S), got=(out, *grads))


def test_relative_attention_without_a_table_and_scale():
    (q, k, v), _, dout, _ = padded_case(torch.bfloat16, 2, 150, 2, 64)
    out = ops().relative_attention(q, k, v)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    check_attention(q, k, v, None, dout, spans=spans_of(2, 150), got=(out, *grads, None))
    other = ops().relative_attention(q * 2, k, v, scale=0.5 / 8)  # (doubling is exact)
    assert torch.equal(other, out)
    # a negative scale is the negative query
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    neg = ops().relative_attention(*x, scale=-0.125)
    gneg = torch.autograd.grad(neg, x, dout)
    y = [(-q).detach().requires_grad_(), k, v]
    pos = ops().relative_attention(*y)
    gpos = torch.autograd.grad(pos, y, dout)
    check_attention(y[0], k, v, None, dout, spans=spans_of(2, 150), got=(neg, -gneg[0], gneg[1], gneg[2], None))
    check_attention(y[0], k, v, None, dout, spans=spans_of(2, 150), got=(pos, *gpos, None))


def test_relative_attention_extreme_scores():
    """Masks of the lowest value inside the table, one-sided tables, and rows that attend to one key only."""
    (q, k, v), bias, dout, _ = padded_case(torch.float16, 1, 300, 2, 64, bias_dtype=torch.float32)
    with torch.no_grad():
        bias[16:] = torch.finfo(torch.float32).min  # no key behind the query
    out = ops().relative_attention(q, k, v, bias)
    grads = torch.autograd.grad(out, (q, k, v, bias), dout)
    u, _ = half_step(torch.float16)
    assert ((out[0, 0] - v[0, 0]).abs() <= 2 * u * v[0, 0].abs()).all()  # the first query sees only itself
    assert all(torch.isfinite(t).all() for t in grads) and grads[3][16:].abs().max() == 0
    with torch.no_grad():
        bias[16:] = -math.inf
    assert torch.equal(ops().relative_attention(q, k, v, bias), out)
    with torch.no_grad():
        bias.fill_(3e4)  # a common shift changes nothing but the last digits of the scores
    shifted = ops().relative_attention(q, k, v, bias)
    plain = ops().relative_attention(q, k, v)
    assert torch.isfinite(shifted).all() and (shifted - plain).abs().max() < 0.05


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [70, 128, 300])
@pytest.mark.parametrize("p,with_ids", [(0.2, False), (0.2, True), (0.99, True)])
def test_relative_attention_dropout(dtype, S, p, with_ids):
    from pytorch_distributed_training_amd.ops.fused import RngKey

    B, A, site = 2, 2, 12
    (q, k, v), bias, dout, valid = padded_case(dtype, B, S, A, 64, lens=[S, S // 2], seed=S)
    rng = RngKey(torch.tensor([99, 3], dtype=torch.int64, device="cuda"), 5,
                 torch.tensor([41, 7], dtype=torch.int32, device="cuda") if with_ids else None)
    out = ops().relative_attention(q, k, v, bias, key_mask=valid, dropout_p=p, rng=rng, site=site)
    grads = torch.autograd.grad(out, (q, k, v, bias), dout)
    keep = keep_mask(rng, p, site, B, A, S)
    assert abs(keep.double().mean().item() - (1 - p)) < 0.01
    check_attention(q, k, v, bias, dout, valid=valid, spans=spans_of(B, S), keep=keep, p_drop=p, got=(out, *grads))


def test_relative_attention_gradients_by_differences():
    """Directional derivative of sum(out * dout) from two forward passes.  A step of 2^-4 along a direction of unit-size
    entries leaves a truncation error of third order, (2^-4)^2 / 6 of the third derivative, and the 16-bit roundings of the
    outputs; both stay below 4 % of the derivative along the gradient itself, which is what is compared."""
    (q, k, v), bias, dout, _ = padded_case(torch.float16, 1, 80, 2, 64, bias_dtype=torch.float32, seed=5)
    out = ops().relative_attention(q, k, v, bias)
    grads = torch.autograd.grad(out, (q, k, v, bias), dout)
    for i, g in enumerate(grads):
        h = 2.0 ** -4 / g.double().pow(2).mean().sqrt()
        vals = []
        for sign in (1, -1):
            args = [t.detach() for t in (q, k, v, bias)]
            args[i] = (args[i].double() + sign * h * g.double()).to(args[i].dtype)
            vals.append(((ops().relative_attention(*args).double() * dout.double()).sum(), args[i].double()))
        step = vals[0][1] - vals[1][1]
        want = (step * g.double()).sum()
        assert abs((vals[0][0] - vals[1][0] - want) / want) < 0.04


def test_relative_attention_layouts_alignment_and_broadcasts():
    B, S, A, D = 2, 90, 3, 64
    (q, k, v), bias, dout, _ = padded_case(torch.bfloat16, B, S, A, D)
    want = ops().relative_attention(q, k, v, bias)
    ref = torch.autograd.grad(want, (q, k, v, bias), dout)
    layouts = {
        "head first": lambda t: t.detach().transpose(1, 2).contiguous().transpose(1, 2),
        "sequence first": lambda t: t.detach().transpose(0, 1).contiguous().transpose(0, 1),
        "odd rows": lambda t: torch.nn.functional.pad(t.detach(), (0, 3))[..., :D],
        "inner stride": lambda t: t.detach().repeat_interleave(2, -1)[..., ::2],
        "off the 16-byte grid": lambda t: torch.cat([t.detach().reshape(-1)[:1], t.detach().reshape(-1)])[1:].view(t.shape),
    }
    for name, make in layouts.items():
        x = [make(t).requires_grad_() for t in (q, k, v)]
        out = ops().relative_attention(*x, bias)
        assert torch.equal(out, want), name
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (*x, bias), make(dout)), ref)), name
    # one key / value head for all, as an expanded view: autograd sums its gradient over the heads
    k1, v1 = (t.detach()[:, :, :1].clone().requires_grad_() for t in (k, v))
    out = ops().relative_attention(q, k1.expand(-1, -1, A, -1), v1.expand(-1, -1, A, -1), bias)
    full = [t.detach().expand(-1, -1, A, -1).contiguous().requires_grad_() for t in (k1, v1)]
    out2 = ops().relative_attention(q, *full, bias)
    assert torch.equal(out, out2)
    a, b = torch.autograd.grad(out, (k1, v1), dout), torch.autograd.grad(out2, full, dout)
    for x, y in zip(a, b):
        torch.testing.assert_close(x, y.sum(2, keepdim=True), rtol=2 ** -7, atol=2 ** -7 * float(y.abs().max()))
    # an expanded output gradient
    g = torch.autograd.grad(ops().relative_attention(q, k, v, bias).sum(), q)[0]
    assert torch.equal(g, torch.autograd.grad(ops().relative_attention(q, k, v, bias), q, torch.ones_like(want))[0])


def test_relative_attention_is_repeatable_and_empty_batches_pass():
    (q, k, v), bias, dout, valid = padded_case(torch.float16, 3, 333, 4, 64, lens=[333, 100, 200], holes=True)
    runs = []
    for _ in range(3):
        out = ops().relative_attention(q, k, v, bias, key_mask=valid)
        runs.append((out, *torch.autograd.grad(out, (q, k, v, bias), dout)))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))
    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        x = [torch.zeros(shape, device="cuda", dtype=torch.float16, requires_grad=True) for _ in range(3)]
        out = ops().relative_attention(*x, bias[:, :2].detach().requires_grad_())
        assert out.shape == shape
        out.sum().backward()
        assert x[0].grad.shape == shape
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")  # rows, but no sequences
    x = [torch.ones(4, 2, 64, device="cuda", dtype=torch.float16, requires_grad=True) for _ in range(3)]
    b2 = bias[:, :2].detach().requires_grad_()
    out = ops().relative_attention(*x, b2, cu_seqlens=cu, max_seqlen=1)
    gs = torch.autograd.grad(out.sum(), (*x, b2))
    assert out.abs().sum() == 0 and all(g.abs().sum() == 0 for g in gs)


def test_relative_attention_on_another_stream_and_in_a_graph():
    (q, k, v), bias, dout, valid = padded_case(torch.float16, 2, 200, 2, 64, lens=[200, 77])

    def step(q, k, v, bias, dout, valid):
        out = ops().relative_attention(q, k, v, bias, key_mask=valid)
        return (out, *torch.autograd.grad(out, (q, k, v, bias), dout))

    want = step(q, k, v, bias, dout, valid)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(q, k, v, bias, dout, valid)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # two captured graphs with their own leaves, replayed in turn, eager work between the replays
    graphs = []
    for shift in (0.0, 0.5):
        args = [(t.detach() + shift).requires_grad_() for t in (q, k, v, bias)] + [dout.clone(), valid.clone()]
        want = step(*args)
        with torch.cuda.stream(side):
            step(*args)
        torch.cuda.synchronize()
        del want
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            res = step(*args)
        graphs.append((g, args, res))
    for turn in range(3):
        for g, args, res in graphs:
            with torch.no_grad():
                args[0].mul_(-1.25)
                args[4].add_(0.125)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, step(*[a.detach().requires_grad_() if i < 4 else a for i, a in enumerate(args)])))


def test_relative_attention_far_offsets():
    """Rows so far apart that their offsets pass 32 bits."""
    S, A, D = 300, 1, 64
    pitch = (1 << 23) - 8  # elements from row to row: 300 rows span 5 GB
    store = torch.empty(S * pitch + D, dtype=torch.float16, device="cuda")
    (q, k, v), bias, dout, _ = padded_case(torch.float16, 1, S, A, D)
    far = []
    for i, t in enumerate((q, k, v)):
        x = store.as_strided((1, S, A, D), (S * pitch, pitch, D, 1), storage_offset=i * 64)
        x.copy_(t.detach())
        far.append(x.detach())
    far = [x.requires_grad_() for x in far]
    out = ops().relative_attention(*far, bias)
    want = ops().relative_attention(q, k, v, bias)
    assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (*far, bias), dout), torch.autograd.grad(want, (q, k, v, bias), dout)))


# ------------------------------------------------------------------------------------------------------ norm + rotation
def check_rope(x, w, cos, sin, pos, interleaved, dy, got, got_dx=None, got_dw=None, eps=1e-6):
    """One side in 64 bits.  y: one rounding on top of fp32 arithmetic on a pair; dx likewise; dw: fp32 sums over all rows."""
    u, tiny = half_step(x.dtype)
    D = x.shape[-1]
    xd = x.detach().double().requires_grad_()
    wd = w.detach().double().requires_grad_() if w is not None else None
    y = xd if wd is None else xd / torch.sqrt(xd.square().mean(-1, keepdim=True) + eps) * wd
    size = y.detach().abs()
    if cos is not None:
        n = 2 * cos.shape[1]
        turn = torch.complex(cos.double(), sin.double())[pos.clamp(0, cos.shape[0] - 1)].unsqueeze(-2)
        pairs = y[..., :n].unflatten(-1, (n // 2, 2) if interleaved else (2, n // 2))
        axis = -1 if interleaved else -2
        z = torch.complex(pairs.select(axis, 0), pairs.select(axis, 1)) * turn
        y = torch.cat((torch.stack((z.real, z.imag), dim=axis).flatten(-2), y[..., n:]), -1)
        both = size[..., :n].unflatten(-1, (n // 2, 2) if interleaved else (2, n // 2)).sum(axis, keepdim=True)
        both = both.expand(*size.shape[:-1], *((n // 2, 2) if interleaved else (2, n // 2))).flatten(-2)
        size = torch.cat((both, size[..., n:]), -1)
    assert ((got.double() - y).abs() <= u * y.abs() + 1e-6 * size + tiny).all()
    if got_dx is None:
        return
    ins = (xd,) if wd is None else (xd, wd)
    grads = torch.autograd.grad(y, ins, dy.double())
    dx = grads[0]
    # each element subtracts a mean over the head: fp32 errors are relative to the head's largest terms
    r = 1.0 if wd is None else (1 / torch.sqrt(xd.detach().square().mean(-1, keepdim=True) + eps)) * wd.detach().abs().amax()
    noise = 4e-6 * r * dy.double().abs().amax(-1, keepdim=True) * (1 + (xd.detach().abs() * r))
    assert ((got_dx.double() - dx).abs() <= u * dx.abs() + noise + tiny).all()
    if wd is not None:
        terms = (dy.double().abs().amax(-1, keepdim=True) * 2 * (xd.detach().abs() * r / wd.detach().abs().amax())).flatten(0, -2).sum(0)
        ub = half_step(w.dtype)[0]
        assert ((got_dw.double() - grads[1]).abs() <= ub * grads[1].abs() + 2e-6 * terms + half_step(w.dtype)[1]).all()


ROPE_SHAPES = [  # leading shape, heads of q and k, dim, rotated, interleaved
    ((1,), 1, 1, 64, 64, False), ((17,), 12, 12, 64, 64, False), ((2, 33), 16, 4, 64, 32, False), ((5, 7), 3, 5, 128, 128, False),
    ((65,), 2, 2, 32, 32, True), ((3, 11), 7, 1, 80, 80, False), ((40,), 4, 4, 72, 24, True), ((9,), 20, 20, 8, 8, True),
    ((130,), 5, 3, 256, 64, False), ((1000,), 1, 2, 96, 96, True), ((31,), 6, 6, 200, 16, False), ((513,), 16, 16, 64, 0, False),
    ((2049,), 2, 1, 16, 16, False)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("lead,hq,hk,D,R,interleaved", ROPE_SHAPES)
def test_qk_norm_rope(dtype, normed, lead, hq, hk, D, R, interleaved):
    if not normed and R == 0:
        pytest.skip("neither norm nor rotation")
    gen = torch.Generator(device="cuda").manual_seed(D + R + hq)

    def normal(*shape, m=0.0, s=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * s + m)

    both = normal(*lead, hq + hk, D, s=1.5).to(dtype)
    q, k = both[..., :hq, :].requires_grad_(), both[..., hq:, :].requires_grad_()
    wdt = torch.float32 if hq % 2 else dtype
    wq, wk = (normal(D, m=1.0, s=0.3).to(wdt).requires_grad_() if normed else None for _ in range(2))
    tokens = math.prod(lead)
    rope = ops().rotary_table(max(700, lead[-1]), R) if R else None  # (default positions need a row each)
    pos = torch.randint(-5, 720, lead, generator=gen, device="cuda") if R and tokens % 2 else None
    out = ops().qk_norm_rope(q, k, wq, wk, rope=rope, positions=pos, interleaved=interleaved)
    douts = [normal(*lead, h, D, s=0.2).to(dtype) for h in (hq, hk)]
    ins = (q, k) + ((wq, wk) if normed else ())
    if pos is None:
        pos = torch.arange(lead[-1], device="cuda").expand(lead)
    grads = torch.autograd.grad(out, ins, douts)
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        check_rope(x, w, *(rope or (None, None)), pos, interleaved, douts[i], out[i], grads[i], grads[2 + i] if normed else None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_qk_norm_rope_large_batch_weight_gradient_and_repeat(dtype):
    """More workgroups than partial rows: the token loop runs several times; the sums keep one order."""
    T, A, D = 70001, 3, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(T, 3, A, D, generator=gen, device="cuda").to(dtype)
    q, k = qkv[:, 0].requires_grad_(), qkv[:, 1].requires_grad_()
    w = [torch.randn(D, generator=gen, device="cuda").add(1).requires_grad_() for _ in range(2)]
    rope = ops().rotary_table(65536, D)
    pos = torch.randint(0, 65536, (T,), generator=gen, device="cuda")
    douts = [torch.randn(T, A, D, generator=gen, device="cuda").to(dtype) for _ in range(2)]
    runs = []
    for _ in range(2):
        out = ops().qk_norm_rope(q, k, *w, rope=rope, positions=pos)
        runs.append((*out, *torch.autograd.grad(out, (q, k, *w), douts)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    for i, x in enumerate((q, k)):
        check_rope(x, w[i], *rope, pos, False, douts[i], runs[0][i], runs[0][2 + i], runs[0][4 + i])


def test_qk_norm_rope_layouts():
    B, S, A, D = 3, 21, 4, 64
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, k = (torch.randn(B, S, A, D, generator=gen, device="cuda").bfloat16() for _ in range(2))
    w = [torch.randn(D, generator=gen, device="cuda").add(1).bfloat16() for _ in range(2)]
    rope = ops().rotary_table(S, D)
    dout = [torch.randn(B, S, A, D, generator=gen, device="cuda").bfloat16() for _ in range(2)]
    ref = None
    for make in (lambda t: t.clone(), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: torch.nn.functional.pad(t, (0, 1))[..., :D], lambda t: t.repeat_interleave(2, -1)[..., ::2]):
        x = [make(t).requires_grad_() for t in (q, k)]
        ww = [t.clone().requires_grad_() for t in w]
        out = ops().qk_norm_rope(*x, *ww, rope=rope)
        res = (*out, *torch.autograd.grad(out, (*x, *ww), [make(t) for t in dout]))
        ref = ref or res
        assert all(torch.equal(a, b) for a, b in zip(ref, res))
    # only one of the two outputs is used
    x = [t.clone().requires_grad_() for t in (q, k)]
    out = ops().qk_norm_rope(*x, *w, rope=rope)
    gq, gk = torch.autograd.grad(out[0], x, dout[0])
    assert torch.equal(gq, ref[2]) and gk.abs().max() == 0
    empty = torch.empty(0, A, D, device="cuda", dtype=torch.float16, requires_grad=True)
    we = [t.half().clone().requires_grad_() for t in w]
    out = ops().qk_norm_rope(empty, empty, *we, rope=rope)
    gs = torch.autograd.grad(out[0].sum() + out[1].sum(), (empty, *we))
    assert out[0].shape == (0, A, D) and all(g.abs().sum() == 0 for g in gs[1:])


def test_rotated_attention_depends_on_relative_positions_only():
    """The two operators together, as a layer uses them: all positions shifted by the same amount give the same output up to
    the roundings of the rotated rows (u each for q' and k', so at most 2 u sum|q'||k'| scale per score)."""
    A, D, S = 2, 64, 150
    gen = torch.Generator(device="cuda").manual_seed(9)
    qkv = torch.randn(1, S, 3, A, D, generator=gen, device="cuda").half()
    w = [torch.ones(D, device="cuda") for _ in range(2)]
    bias = torch.randn(32, A, generator=gen, device="cuda")
    rope = ops().rotary_table(5000, D)
    outs = []
    for shift in (0, 4000):
        q, k = ops().qk_norm_rope(qkv[:, :, 0], qkv[:, :, 1], *w, rope=rope, positions=torch.arange(S, device="cuda")[None] + shift)
        outs.append(ops().relative_attention(q, k, qkv[:, :, 2], bias).double())
    # |q'| = |k'| = 8: a score moves by at most 2 u * 64 / 8, a probability by a factor e^(2 * that), the output rounds twice
    u, _ = half_step(torch.float16)
    top = qkv[:, :, 2].double().abs().max()
    assert (outs[0] - outs[1]).abs().max() <= 2 * (math.exp(4 * 16 * u) - 1) * top + 6 * u * top


@pytest.mark.parametrize("dtype", DTYPES)
def test_relative_attention_far_buckets_give_back_the_rounding_of_p(dtype):
    """Scores of two levels, whose probabilities round the same way in every row, and values that follow them: the forward's
    output is off by the same e = u p / (1 + p) in every row (p = 0.5 (1 + 0.9 u) is stored as 0.5).  Without giving it back,
    the far buckets would add up e times their share of the row over all rows, S e / 2 each; what may remain is the share of
    the keys that lie in a far bucket but not in chunks that are far as a whole: the buckets' ends, the workgroup's rows and two
    chunks, in all no more than 64 + 128 + 2 * 64 keys on a side."""
    S, u = 2048, half_step(dtype)[0]
    p = 0.5 * (1 + 0.9 * u)
    q = torch.zeros(1, S, 1, 64, dtype=dtype, device="cuda")
    k, v, dout = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    q[..., :3] = 1
    left = math.log(p) * 8  # the scale is 1 / 8; the score in three parts, each of the dtype
    for i in range(3):
        part = torch.tensor(left, dtype=torch.float64).to(dtype)
        k[:, 1::2, :, i] = part
        left -= float(part)
    v[:, 0::2, :, 5] = 1
    v[:, 1::2, :, 5] = -1
    dout[..., 5] = 1
    bias = torch.zeros(32, 1, device="cuda", requires_grad=True)
    for t in (q, k, v):
        t.requires_grad_()
    ops().relative_attention(q, k, v, bias, max_distance=128).backward(dout)
    score = (q.detach().double()[0, :, 0] @ k.detach().double()[0, :, 0].T) / 8
    prob = score.softmax(-1)
    dp = torch.ones(S, 1, dtype=torch.float64, device="cuda") * v.detach().double()[0, :, 0, 5]
    ds = prob * (dp - (prob * dp).sum(-1, keepdim=True))
    gap = torch.arange(S, device="cuda")
    bucket = bucket_rule(gap[None, :] - gap[:, None], 32, 128)
    true = torch.zeros(32, dtype=torch.float64, device="cuda").index_add_(0, bucket.flatten(), ds.flatten())
    e = 0.45 * u / (1 + p)
    for b in (15, 31):
        off = abs(float(bias.grad[b, 0]) - float(true[b]))
        left_over = S * e * (64 + 128 + 2 * 64) / S * 1.05 + F32 * S  # (1.05: the keys of either level)
        assert off < left_over, (b, off, left_over, S * e / 2)
        assert dtype == torch.float16 or left_over < 0.4 * S * e


@pytest.mark.parametrize("form", ["short mask", "long mask", "packed"])
def test_captured_passes_read_the_lengths_and_masks_of_each_replay(form):
    """A captured training pass with its buffers refilled between replays: other masks, other sequence borders."""
    A, D, T = 2, 64, 400
    S = {"short mask": 100, "long mask": 200, "packed": 0}[form]
    lengths = [[S, 0], [1, S], [S // 2, 65]] if S else [[300, 0, 64], [5, 130, 1], [0, 399, 1]]
    gen = torch.Generator(device="cuda").manual_seed(S)
    shape = (2, S, A, D) if S else (T, A, D)
    q, k, v = ((torch.randn(shape, generator=gen, device="cuda")).half().requires_grad_() for _ in range(3))
    bias = torch.randn(32, A, generator=gen, device="cuda").requires_grad_()
    dout = torch.randn(shape, generator=gen, device="cuda").half()

    def where(lens):
        lens = torch.tensor(lens, device="cuda")
        if S:
            return torch.arange(S, device="cuda")[None, :] < lens[:, None]
        return torch.cat([lens.new_zeros(1), lens.cumsum(0)]).int()

    def step(at):
        more = {"key_mask": at} if S else {"cu_seqlens": at, "max_seqlen": 399}
        out = ops().relative_attention(q, k, v, bias, **more)
        return (out, *torch.autograd.grad(out, (q, k, v, bias), dout))

    held = where(lengths[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = step(held)
    for lens in lengths + lengths[:1]:
        held.copy_(where(lens))
        graph.replay()
        torch.cuda.synchronize()
        want = step(where(lens))
        assert all(torch.equal(a, b) for a, b in zip(res, want)), lens


@pytest.mark.parametrize("S", [60, 300])
def test_relative_attention_of_one_tensor_and_with_a_frozen_table(S):
    """The same tensor as queries, keys and values: its gradient is the sum of the three; a table that takes no gradient."""
    (x, y, z), bias, dout, _ = padded_case(torch.bfloat16, 2, S, 2, 64, seed=S)
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    out = ops().relative_attention(*parts, bias)
    apart = torch.autograd.grad(out, (*parts, bias), dout)
    x = x.detach().clone().requires_grad_()
    frozen = bias.detach()
    same = ops().relative_attention(x, x, x, frozen)
    assert torch.equal(same, out)
    (g,) = torch.autograd.grad(same, x, dout)
    u = half_step(torch.bfloat16)[0]
    total = sum(t.double() for t in apart[:3])
    bound = 2 * u * (apart[0].double().abs() + apart[1].double().abs() + apart[2].double().abs())  # two sums of 16-bit terms
    assert ((g.double() - total).abs() <= bound * (1 + u) + 1e-30).all()


def test_two_calls_at_once_on_two_streams():
    """Calls of both operators on two streams, backward passes included, as eager results one after the other."""
    cases = [padded_case(torch.float16, 2, S, 2, 64, lens=[S, S // 3], seed=S) for S in (120, 450)]
    rope = ops().rotary_table(512, 64)
    w = [(torch.rand(64, device="cuda") + 0.5).requires_grad_() for _ in range(2)]

    def step(case):
        (q, k, v), bias, dout, valid = case
        a, b = ops().qk_norm_rope(q, k, *w, rope=rope)
        out = ops().relative_attention(a, b, v, bias, key_mask=valid)
        return (out, *torch.autograd.grad(out, (q, k, v, bias, *w), dout))

    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step(c))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("limit", [50, 100, 130])
def test_relative_attention_cuts_packed_sequences_at_the_length_announced(limit):
    """Sequences longer than max_seqlen count up to it; rows before the first and behind the last one belong to none."""
    lead, lens, tail, A, D = 3, [20, 150, 1, 131], 9, 2, 64
    T = lead + sum(lens) + tail
    gen = torch.Generator(device="cuda").manual_seed(limit)
    q, k, v = (torch.randn(T, A, D, generator=gen, device="cuda").half().requires_grad_() for _ in range(3))
    bias = torch.randn(32, A, generator=gen, device="cuda").requires_grad_()
    dout = (torch.randn(T, A, D, generator=gen, device="cuda") * 0.25).half()
    cu = torch.tensor([lead] + lens, device="cuda").cumsum(0).int()
    junk = [torch.full((T, A, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(8)]  # (what the outputs' memory held)
    del junk
    out = ops().relative_attention(q, k, v, bias, cu_seqlens=cu, max_seqlen=limit)
    grads = torch.autograd.grad(out, (q, k, v, bias), dout)
    spans = [(lo, min(hi, lo + limit)) for lo, hi in zip(cu.tolist()[:-1], cu.tolist()[1:])]
    check_attention(q, k, v, bias, dout, spans=spans, got=(out, *grads))
    outside = torch.ones(T, dtype=torch.bool, device="cuda")
    for lo, hi in spans:
        outside[lo:hi] = False
    for t in (out, *grads[:3]):
        assert t[outside].abs().sum() == 0
