"""What the position operators' nodes do not know - forward-mode differentiation, traces - is refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

from pytorch_distributed_training_amd.ops import available, qk_norm_rope, relative_attention

pytestmark = pytest.mark.skipif(not available(), reason="the native extension is not built")
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _arguments(device):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 8, 2, 64, generator=g).half().to(device) for _ in range(3))
    return dict(q=q, k=k, v=v), torch.randn(32, 2, generator=g).to(device), [torch.ones(64, device=device) for _ in range(2)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("which", ["q", "k", "v", "bias"])
def test_tangents_of_relative_attention_are_refused(device, which, requires_grad):
    qkv, bias, _ = _arguments(device)
    args = {**qkv, "bias": bias}
    with fwd.dual_level():
        args[which] = fwd.make_dual(args[which].requires_grad_(requires_grad), torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            relative_attention(**args)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["q", "k", "q_weight", "k_weight", "cos"])
def test_tangents_of_qk_norm_rope_are_refused(device, which):
    qkv, _, (wq, wk) = _arguments(device)
    args = dict(q=qkv["q"], k=qkv["k"], q_weight=wq, k_weight=wk, cos=torch.ones(8, 32, device=device))
    with fwd.dual_level():
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        cos = args.pop("cos")
        with pytest.raises(RuntimeError, match="forward-mode"):
            qk_norm_rope(**args, rope=(cos, torch.zeros(8, 32, device=device)))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("trace", [torch.jit.trace, lambda f, x: make_fx(f)(*x), lambda f, x: make_fx(f, tracing_mode="fake")(*x)],
                         ids=["jit", "fx", "fake"])
def test_traces_are_refused(device, trace):
    qkv, bias, w = _arguments(device)
    x = (qkv["q"], qkv["k"], qkv["v"])
    with pytest.raises(RuntimeError, match="traced"):
        trace(lambda q, k, v: relative_attention(q, k, v, bias), x)
    with pytest.raises(RuntimeError, match="traced"):
        trace(lambda q, k, v: qk_norm_rope(q, k, *w)[0], x)


@pytest.mark.gpu
def test_calls_beside_a_dual_level_stay():
    qkv, bias, _ = _arguments("cuda")
    want = relative_attention(**qkv, bias=bias)
    with fwd.dual_level():
        fwd.make_dual(qkv["q"], torch.ones_like(qkv["q"]))  # (another tensor carries the tangent)
        assert torch.equal(relative_attention(**qkv, bias=bias), want)
