"""Arguments of relative_attention at the edges of what its documentation allows."""
import math

import pytest
import torch

from pytorch_distributed_training_amd.ops import relative_attention
from pytorch_distributed_training_amd.ops.attention import mask_bits


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int8, torch.int16, torch.uint8, torch.int32, torch.int64, torch.bool])
@pytest.mark.parametrize("S", [50, 300])
def test_masks_of_every_whole_number_type(dtype, S):
    gen = torch.Generator(device="cuda").manual_seed(S)
    q, k, v = (torch.randn(2, S, 2, 64, generator=gen, device="cuda").half() for _ in range(3))
    valid = torch.rand(2, S, generator=gen, device="cuda") < 0.7
    value = {torch.int8: -128, torch.int16: 256, torch.int32: 1 << 30, torch.int64: 1 << 40, torch.uint8: 128}.get(dtype, 1)
    mask = valid.to(dtype) * value if dtype != torch.bool else valid
    assert torch.equal(relative_attention(q, k, v, key_mask=mask), relative_attention(q, k, v, key_mask=valid))
    assert torch.equal(mask_bits(mask), mask_bits(valid))


def test_complex_masks_are_refused():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="truth values"):
        relative_attention(q, q, q, key_mask=torch.ones(1, 4, dtype=torch.complex64))


@pytest.mark.parametrize("scale", [1e-20, -1e-20, 1e-40, 1e-60, 1e20, -1e30, 1e39, math.nan])
def test_scales_that_fp32_cannot_work_with_are_refused(scale):
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="scale"):
        relative_attention(q, q, q, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("S", [60, 300])
@pytest.mark.parametrize("a,b", [(-30, -33), (20, 20), (-64, 3)])
def test_scales_of_either_end(S, a, b):
    """Powers of two moved between q, k and the scale change no digit of the scores (bf16 and fp32 hold all of them)."""
    gen = torch.Generator(device="cuda").manual_seed(S)
    q, k, v = (torch.randn(2, S, 2, 64, generator=gen, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    bias = torch.randn(32, 2, generator=gen, device="cuda").requires_grad_()
    dout = torch.randn(2, S, 2, 64, generator=gen, device="cuda").bfloat16()
    want = relative_attention(q, k, v, bias, scale=0.125)
    ref = torch.autograd.grad(want, (q, k, v, bias), dout)
    x = [(q.detach().double() * 2.0 ** a).bfloat16().requires_grad_(), (k.detach().double() * 2.0 ** b).bfloat16().requires_grad_(), v, bias]
    out = relative_attention(*x, scale=2.0 ** (-3 - a - b))
    got = torch.autograd.grad(out, x, dout)
    torch.testing.assert_close(out, want, rtol=2 ** -7, atol=1e-6)
    for g, w, e in zip(got, ref, (a, b, 0, 0)):
        d = (g.double() * 2.0 ** e - w.double()).norm() / w.double().norm()
        assert d < 2 ** -8, float(d)


@pytest.mark.gpu
@pytest.mark.parametrize("sign", [1, -1])
def test_the_smallest_scale_leaves_the_table(sign):
    S = 200
    gen = torch.Generator(device="cuda").manual_seed(S)
    q, k, v = (torch.randn(1, S, 2, 64, generator=gen, device="cuda").half() for _ in range(3))
    bias = torch.randn(32, 2, generator=gen, device="cuda") * 5
    a = relative_attention(q, k, v, bias, scale=sign * 2.0 ** -64)
    b = relative_attention(torch.zeros_like(q), k, v, bias)
    assert torch.isfinite(a).all() and (a.float() - b.float()).abs().max() <= 2e-3 * v.abs().max()


@pytest.mark.gpu
def test_generator_states_of_another_device_are_refused():
    from pytorch_distributed_training_amd.ops.fused import RngKey

    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16, device="cuda")
    state = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="rng state|device of q"):
        relative_attention(q, q, q, dropout_p=0.1, rng=RngKey(state.cpu(), 0, None))
    with pytest.raises(RuntimeError, match="device of q"):
        relative_attention(q, q, q, dropout_p=0.1, rng=RngKey(state, 0, torch.zeros(1, dtype=torch.int32)))
    if torch.cuda.device_count() > 1:
        other = RngKey(state.to("cuda:1"), 0, None)
        with pytest.raises(RuntimeError, match="device of q"):
            relative_attention(q, q, q, dropout_p=0.1, rng=other)


@pytest.mark.gpu
def test_weights_tables_positions_and_borders_of_any_layout():
    gen = torch.Generator(device="cuda").manual_seed(0)
    B, S, A, D = 3, 20, 2, 64
    q, k, v = (torch.randn(B, S, A, D, generator=gen, device="cuda").half().requires_grad_() for _ in range(3))
    w = [torch.rand(D, generator=gen, device="cuda").add(0.5).requires_grad_() for _ in range(2)]
    from pytorch_distributed_training_amd.ops import qk_norm_rope, rotary_table

    cos, sin = rotary_table(100, D)
    pos = torch.arange(S, device="cuda")[None] + 5

    def run(w, rope, pos):
        y = qk_norm_rope(q, k, *w, rope=rope, positions=pos)
        return (*y, *torch.autograd.grad(y, (q, k, *w), [torch.ones_like(t) for t in y]))

    want = run(w, (cos, sin), pos.repeat(B, 1))
    spread = [t.detach().repeat_interleave(3)[::3].requires_grad_() for t in w]
    shifted = [torch.cat([t.detach()[:1], t.detach()])[1:].requires_grad_() for t in w]  # (off the 16-byte grid)
    wide = [torch.cat([t, t], 1)[:, :D // 2] for t in (cos, sin)]
    for args in ((w, (cos, sin), pos.expand(B, S)), (spread, (cos, sin), pos.repeat(B, 2)[:, :S]), (shifted, wide, pos.repeat(B, 1)),
                 (w, [torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in (cos, sin)], pos.repeat(B, 1))):
        assert all(torch.equal(a, b) for a, b in zip(run(*args), want))
    rows = [t.detach().reshape(B * S, A, D) for t in (q, k, v)]
    cu = torch.tensor([0, 7, 30, 60], dtype=torch.int32, device="cuda")
    want = relative_attention(*rows, cu_seqlens=cu, max_seqlen=30)
    assert torch.equal(relative_attention(*rows, cu_seqlens=cu.repeat_interleave(2)[::2], max_seqlen=30), want)


@pytest.mark.gpu
def test_more_heads_than_a_launch_holds_are_refused():
    """Expanded rows: the grid of (sample, head) pairs passes 2^32 threads while the output is 270 MB."""
    one = torch.zeros(1, 1, 16, 8, dtype=torch.float16, device="cuda")
    q = one.expand((1 << 20) + 1, 1, 16, 8)
    with pytest.raises(RuntimeError, match="argument check"):
        relative_attention(q, q, q)
    q = one.expand(1 << 19, 1, 16, 8)
    assert relative_attention(q, q, q).abs().max() == 0
