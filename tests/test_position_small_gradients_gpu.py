"""relative_attention in fp16 with output gradients whose products with probabilities lie below fp16's normal numbers.

Roundings are independent and uniform, so a rounding of x contributes (u |x|)^2 / 3 to the expected square of an error, u half a
unit of the dtype; the fp32 sums add nothing that counts.  The gradients' errors, as norms over thousands of elements, are held
to 1.5 times what the roundings of p, ds, and the stored results amount to when ds keeps its relative precision."""
import math

import pytest
import torch

from test_position_ops_gpu import bucket_rule, half_step, keep_mask, ops

pytestmark = pytest.mark.gpu


def reference(q, k, v, bias, dout, scale, max_distance=128, keep=None, p_drop=0.0):
    """Gradients in 64 bits of [S, A, D] rows, and the expected squared error of each element."""
    dtype = q.dtype
    u, tiny = half_step(dtype)
    n = q.shape[0]
    qq, kk, vv, gg = (t.detach().transpose(0, 1).double() for t in (q, k, v, dout))
    place = torch.arange(n, device="cuda")
    bucket = bucket_rule(place[None, :] - place[:, None], bias.shape[0], max_distance)
    s = qq @ kk.transpose(1, 2) * scale + bias.detach().double()[bucket].permute(2, 0, 1)
    P = torch.softmax(s, -1)
    Z = keep.double() / (1 - p_drop) if keep is not None else torch.ones_like(P)
    dP = gg @ vv.transpose(1, 2) * Z
    ds = P * (dP - (P * dP).sum(-1, keepdim=True))
    # delta carries the roundings of the forward's probabilities (relative to 2^8 of the row's running maximum at most, so the
    # absolute part of theirs is 2^-8 tiny and less of the row's sum); then ds is rounded itself
    d_delta = ((P * dP) ** 2).sum(-1, keepdim=True) * u * u / 3
    ds_err = (u * ds) ** 2 / 3 + P * P * d_delta
    out = lambda x: (u * x) ** 2 / 3 + tiny * tiny / 3
    dq, dk, dv = ds @ kk * scale, ds.transpose(1, 2) @ qq * scale, (P * Z).transpose(1, 2) @ gg
    err = [scale ** 2 * (ds_err @ kk ** 2) + out(dq), scale ** 2 * (ds_err.transpose(1, 2) @ qq ** 2) + out(dk),
           ((u * P * Z) ** 2 / 3).transpose(1, 2) @ gg ** 2 + out(dv)]
    db = torch.zeros(bias.shape, dtype=torch.float64, device="cuda")
    db.index_add_(0, bucket.flatten(), ds.flatten(1).t().contiguous())
    return [t.transpose(0, 1) for t in (dq, dk, dv)] + [db], [t.sum() for t in err]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,size", [(60, 1e-4), (128, 1e-4), (128, 0.2), (300, 2e-4), (1000, 1e-3), (1000, 1e-4), (2100, 1e-3), (2100, 3.0)])
def test_gradients_of_small_output_gradients(S, size, D):
    A, scale = 2, 1.0
    gen = torch.Generator(device="cuda").manual_seed(S + D)
    normal = lambda: torch.randn(1, S, A, D, generator=gen, device="cuda")
    q, k, v = ((normal() / math.sqrt(D)).half().requires_grad_(), normal().half().requires_grad_(), normal().half().requires_grad_())
    bias = torch.randn(32, A, generator=gen, device="cuda").requires_grad_()
    dout = (normal() * size).half()
    out = ops().relative_attention(q, k, v, bias, scale=scale)
    got = torch.autograd.grad(out, (q, k, v, bias), dout)
    want, err = reference(q[0], k[0], v[0], bias, dout[0], scale)
    for name, g, w, e in zip(("dq", "dk", "dv"), got, want, err):
        off = (g[0].double() - w).norm()
        assert off <= 1.5 * e.sqrt(), (name, float(off / w.norm()), float(e.sqrt() / w.norm()))
    assert ((got[3].double() - want[3]).norm() / want[3].norm()).item() < 5e-3


@pytest.mark.parametrize("S", [100, 500])
@pytest.mark.parametrize("p", [0.1, 0.99])
def test_small_output_gradients_under_dropout(S, p):
    from pytorch_distributed_training_amd.ops.fused import RngKey

    A, D, site, scale = 2, 64, 3, 1.0
    gen = torch.Generator(device="cuda").manual_seed(S)
    normal = lambda: torch.randn(1, S, A, D, generator=gen, device="cuda")
    q, k, v = ((normal() / math.sqrt(D)).half().requires_grad_(), normal().half().requires_grad_(), normal().half().requires_grad_())
    bias = torch.randn(32, A, generator=gen, device="cuda").requires_grad_()
    dout = (normal() * 2e-4).half()
    rng = RngKey(torch.tensor([5, 6], dtype=torch.int64, device="cuda"), 1, None)
    out = ops().relative_attention(q, k, v, bias, scale=scale, dropout_p=p, rng=rng, site=site)
    got = torch.autograd.grad(out, (q, k, v, bias), dout)
    want, err = reference(q[0], k[0], v[0], bias, dout[0], scale, keep=keep_mask(rng, p, site, 1, A, S)[0], p_drop=p)
    for name, g, w, e in zip(("dq", "dk", "dv"), got, want, err):
        off = (g[0].double() - w).norm()
        assert off <= 1.5 * e.sqrt(), (name, float(off / w.norm()), float(e.sqrt() / w.norm()))


@pytest.mark.parametrize("lens", [[70, 0, 1, 128, 30], [700, 5, 300]])
def test_small_and_large_sequences_of_a_packed_batch(lens):
    """Every sequence of a packed batch by its own gradients: the same results as alone, whatever its neighbours carry."""
    A, D, T = 2, 64, sum(lens)
    gen = torch.Generator(device="cuda").manual_seed(T)
    q, k, v = (torch.randn(T, A, D, generator=gen, device="cuda").half().requires_grad_() for _ in range(3))
    bias = torch.randn(32, A, generator=gen, device="cuda").requires_grad_()
    dout = torch.randn(T, A, D, generator=gen, device="cuda")
    edges = torch.tensor([0] + lens).cumsum(0).tolist()
    for i, (lo, hi) in enumerate(zip(edges[:-1], edges[1:])):
        dout[lo:hi] *= [1e-4, 1.0, 0.0, 3e-3, 200.0][i]
    dout = dout.half()
    cu = torch.tensor(edges, dtype=torch.int32, device="cuda")
    got = torch.autograd.grad(ops().relative_attention(q, k, v, bias, cu_seqlens=cu, max_seqlen=max(lens)), (q, k, v), dout)
    for lo, hi in zip(edges[:-1], edges[1:]):
        if hi == lo:
            continue
        x = [t.detach()[None, lo:hi].clone().requires_grad_() for t in (q, k, v)]
        if max(lens) > 128 and hi - lo <= 128:  # (alone they would take the short kernel)
            want, err = reference(x[0][0], x[1][0], x[2][0], bias, dout[lo:hi], D ** -0.5)
            for g, w, e in zip(got, want, err):
                assert (g[lo:hi].double() - w).norm() <= 1.5 * e.sqrt() + 1e-30
            continue
        alone = torch.autograd.grad(ops().relative_attention(*x, bias), x, dout[None, lo:hi])
        assert all(torch.equal(a[0], g[lo:hi]) for a, g in zip(alone, got))


@pytest.mark.parametrize("S", [100, 600])
def test_lifted_products_do_not_overflow(S):
    """Values near 1000 beside output gradients of 1e-3 and less, gradients at both ends of fp16, and rows of zeros."""
    gen = torch.Generator(device="cuda").manual_seed(S)
    normal = lambda: torch.randn(1, S, 2, 64, generator=gen, device="cuda")
    q, k = (normal().half().requires_grad_() for _ in range(2))
    bias = torch.randn(32, 2, generator=gen, device="cuda").requires_grad_()
    for values, size in ((1000.0, 1e-3), (1000.0, 6e-8), (1.0, 6e4), (1.0, 0.0), (30.0, 1e-5)):
        v = (normal() * values).half().requires_grad_()
        dout = (normal().clamp(-1, 1) * size).half()
        got = torch.autograd.grad(ops().relative_attention(q, k, v, bias), (q, k, v, bias), dout)
        if size < 1e4:
            assert all(torch.isfinite(t).all() for t in got), (values, size)
        if size == 0.0:
            assert all(t.abs().max() == 0 for t in got)
        want, err = reference(q[0], k[0], v[0], bias, dout[0], 0.125)
        if size < 1e4:
            for g, w, e in zip(got, want, err):
                assert (g[0].double() - w).norm() <= 1.5 * e.sqrt() + 1e-30, (values, size)
