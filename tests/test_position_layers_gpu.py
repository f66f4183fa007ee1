"""Encoder layers with position options beyond the lengths of the short backward kernel: training, dropout rows."""
import copy

import pytest
import torch

from test_position_model_gpu import OPTIONS, _batch, _pack, _pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("S", [900, 513])
def test_long_samples_draw_their_own_masks(S, packed):
    """Training with dropout beyond 512 tokens: the masks of a sample are the same alone, in a batch, padded and packed, and
    neighbouring sample ids do not share them (the loss of the same text under another id differs)."""
    from pytorch_distributed_training_amd.models.bert import build_model
    from pytorch_distributed_training_amd.ops.arena import ParamArena

    torch.manual_seed(0)
    model = build_model("bert-tiny", max_position_embeddings=1024, **OPTIONS["all"]).cuda()
    arena = ParamArena(model, torch.device("cuda"), torch.float16)
    model.enable_native(arena, seed=3)
    model.train()
    batch = _batch(model.config, S=S, lens=[S, S - 70, 40])
    form = _pack if packed else (lambda b: b)

    def run(b, ids):
        arena.zero_grad()
        arena.window = 7
        out = model(**form(b), sample_ids=torch.tensor(ids, device="cuda"))
        (out.loss * 64).backward()
        return out.logits.detach().clone(), arena.grad.clone()

    logits, grad = run(batch, [5, 6, 2])
    again, grad2 = run(batch, [5, 6, 2])
    assert torch.equal(logits, again) and torch.equal(grad, grad2) and torch.isfinite(grad).all()
    for i, sid in enumerate((5, 6, 2)):
        alone, _ = run({k: v[i:i + 1] for k, v in batch.items()}, [sid])
        torch.testing.assert_close(alone, logits[i:i + 1], rtol=5e-3, atol=5e-3)
    other, _ = run(batch, [6, 5, 3])
    assert (other - logits).abs().amax(1).min() > 1e-4
    packed = not packed
    form = _pack if packed else (lambda b: b)
    logits2, grad3 = run(batch, [5, 6, 2])
    torch.testing.assert_close(logits2, logits, rtol=5e-3, atol=5e-3)
    assert ((grad - grad3).norm() / grad.norm()).item() < 2e-2


@pytest.mark.parametrize("option", ["bias", "all"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("S", [200, 400])
@pytest.mark.parametrize("packed", [False, True])
def test_long_layers_train_like_the_torch_path(option, dtype, S, packed):
    """The comparison and the tolerances of the short lengths, where the long kernels run: strides of the fused projection,
    chunks beyond the last bucket."""
    ref, nat, arena = _pair("bert-tiny", dtype, max_position_embeddings=512, **OPTIONS[option])
    batch = _batch(ref.config, S=S, lens=[S, S - 7, S // 2, 3])
    ref.train(); nat.train()
    o_ref = ref(**batch)
    o_nat = nat(**(_pack(batch) if packed else batch))
    tol = 3e-2 if dtype == torch.bfloat16 else 5e-3
    torch.testing.assert_close(o_nat.logits, o_ref.logits, rtol=tol, atol=tol)
    o_ref.loss.backward()
    arena.zero_grad()
    o_nat.loss.backward()
    named = dict(nat.named_parameters())
    for n, p in ref.named_parameters():
        g_ref, g_nat = p.grad.float(), named[n].grad.float()
        if g_ref.norm().item() < 1e-8:
            assert g_nat.norm().item() < 1e-4, n
            continue
        if n == "classifier.bias":
            # the mean over the samples of softmax(logits) - onehot, whose norm may be small: where each of two logits may be off by
            # d = tol (1 + |logit|), either class's probability is off by p (1 - p) 2 d <= d / 2
            off = 0.5 * tol * (1 + o_ref.logits.abs().amax().item())
            assert (g_nat - g_ref).abs().max().item() <= off, n
            continue
        assert ((g_nat - g_ref).norm() / g_ref.norm()).item() < (8e-2 if dtype == torch.bfloat16 else 2e-2), n
    first = arena.grad.clone()
    nat(**(_pack(batch) if packed else batch)).loss.backward()
    torch.testing.assert_close(arena.grad, 2 * first, rtol=1e-3, atol=1e-6)


@pytest.mark.parametrize("nodes", ["0", "1"])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("S", [300, 400])
def test_layer_gradients_do_not_carry_the_rounding_of_the_output(S, packed, nodes, monkeypatch):
    """Keys and values with a common offset of 16.  The gradient of the scores, p (dp - delta), does not see it, but an error e
    of a row's delta gives its dq the error scale e sum_j p_j k_j = e 16 / 8 in every element.

    delta from the rounded output: outputs near 16 are stored in steps of 2^-6, off by 2^-6 / sqrt(12) = 0.0045; over the 64
    elements of a row of unit output gradients e = 8 * 0.0045 = 0.036, and dq is off by 0.072.
    What an exact output leaves is the rounding of the forward's p, independent from key to key: with sum_j p_j^2 = r^2 it is
    e = (u / sqrt(3)) r 16 * 8 = 0.036 r (u = 2^-11), and dq is off by 0.072 r.
    dq itself: values and keys spread by 0.7 (weights of 0.06 over 128 inputs), so dp spreads by 8 * 0.7 = 5.5 and
    |dq| = r 5.5 * 0.7 / 8 = 0.48 r in an element.  The second is therefore 0.15 of dq whatever r is; the first is 0.15 / r, more
    than all of dq for r = 0.12 (300 keys whose scores spread by one, r^2 = e / 300 or a little more).  The roundings of q, k
    and v (steps of 2^-6 beside a spread of 0.7: 0.007) and of the layers' other tensors are small beside that; 0.25 leaves
    them room.  (Without the output's low part: 0.94 and 1.05 at 300 and 400 keys.)"""
    monkeypatch.setenv("PDT_LAYER_NODES", nodes)
    ref, nat, arena = _pair("bert-tiny", torch.float16, max_position_embeddings=512, num_hidden_layers=2, **OPTIONS["bias"])
    offset = 16.0
    with torch.no_grad():
        for lyr in ref.bert.encoder.layers():
            sa, out = lyr.attention.self, lyr.attention.output.dense
            sa.key.bias += offset
            sa.value.bias += offset
            out.bias -= out.weight.sum(1) * offset  # (what follows the attention does not see the offset)
    from pytorch_distributed_training_amd.models.bert import MaskInfo
    from pytorch_distributed_training_amd.ops import fused
    from pytorch_distributed_training_amd.ops.arena import ParamArena

    nat = copy.deepcopy(ref)
    arena = ParamArena(nat, torch.device("cuda"), torch.float16)
    nat.enable_native(arena, seed=1)
    ref.train(); nat.train()
    gen = torch.Generator(device="cuda").manual_seed(S)
    B, H = 2, ref.config.hidden_size
    x = torch.randn(B, S, H, generator=gen, device="cuda").half()
    dy = torch.randn(B, S, H, generator=gen, device="cuda").half()
    xr, mask = x.float(), MaskInfo(torch.ones(B, S, dtype=torch.int32, device="cuda"), B, S, x.device)
    for lyr in ref.bert.encoder.layers():
        xr = lyr._forward_torch(xr, mask)
    xr.backward(dy.float())
    arena.zero_grad()
    if packed:
        cu = torch.tensor([0, S, 2 * S], dtype=torch.int32, device="cuda")
        m = MaskInfo(None, B, S, x.device, cu_seqlens=cu, rowmap=torch.arange(B * S, dtype=torch.int32, device="cuda"))
        xn, dn = x.view(B * S, H), dy.view(B * S, H)
    else:
        m, xn, dn = mask, x, dy
    nat.runtime.begin_forward(None)
    fused.encoder_stack_forward(nat.bert.encoder.layers(), xn.clone().requires_grad_(), m).backward(dn)
    named = dict(nat.named_parameters())
    for n, p in ref.named_parameters():
        if n.endswith(("self.query.weight", "self.query.bias", "relative_attention_bias.weight")):
            err = ((named[n].grad.float() - p.grad).norm() / p.grad.norm()).item()
            assert err < 0.25, (n, err)


@pytest.mark.parametrize("S,positions", [(64, 512), (200, 512), (600, 1024)])
def test_graphed_steps_of_position_models_match_eager(S, positions):
    """Captured training steps, replayed, against eager ones (the tolerance of the same test without position options); with
    dropout every replay draws new masks."""
    from pytorch_distributed_training_amd.data.synthetic import fixed_batch
    from pytorch_distributed_training_amd.engine import Engine
    from pytorch_distributed_training_amd.models.bert import build_model
    from pytorch_distributed_training_amd.optim import AdamW
    from pytorch_distributed_training_amd.utils.graph import GraphedStep

    def run(graphed, name, lr, steps):
        torch.manual_seed(3)
        eng = Engine(fp16=True, seed=11, init_scale=1024.0)
        model = build_model(name, max_position_embeddings=positions, **OPTIONS["all"])
        opt = AdamW(params=model.parameters(), lr=lr)
        model, opt = eng.prepare(model, opt)
        model.train()
        batches = [fixed_batch(4, S, eng.unwrap_model(model).config.vocab_size, eng.device, seed=50 + i) for i in range(2)]
        step = GraphedStep(eng, model, opt, warmup=2) if graphed else None
        losses = []
        for i in range(steps):
            if graphed:
                losses.append(float(step(batches[i % 2]).item()))
                continue
            out = model(**batches[i % 2])
            eng.backward(out.loss)
            opt.step()
            opt.zero_grad()
            losses.append(float(out.loss.item()))
        return losses

    eager, graphed = run(False, "bert-tiny-nodrop", 1e-3, 7), run(True, "bert-tiny-nodrop", 1e-3, 7)
    assert max(abs(a - b) for a, b in zip(eager, graphed)) < 2e-3, (eager, graphed)
    same = run(True, "bert-tiny", 0.0, 8)[3::2]  # replays of one batch at learning rate 0: only the masks change
    assert len(set(same)) == len(same), same


@pytest.mark.parametrize("S", [64, 200])
def test_windows_on_several_streams_add_up_the_same_gradients(S, monkeypatch):
    """Forward passes of the next micro-batch overlap the backward of the last one: the window's gradients are those of the
    micro-batches one after the other, up to the order of two additions per element."""
    from pytorch_distributed_training_amd.engine import Engine
    from pytorch_distributed_training_amd.models.bert import build_model
    from pytorch_distributed_training_amd.optim import AdamW

    grads = []
    for overlap in ("1", "0"):
        monkeypatch.setenv("PDT_OVERLAP_MICRO", overlap)
        torch.manual_seed(0)
        eng = Engine(fp16=True, seed=1, init_scale=64.0)
        model = build_model("bert-tiny", max_position_embeddings=512, **OPTIONS["all"])
        model, opt = eng.prepare(model, AdamW(params=model.parameters(), lr=0.0))[:2]
        inner = getattr(model, "module", model)
        model.train()
        batches = []
        for i, lens in enumerate(([S, S - 7, 3, 40], [S // 2, S, 1, 9], [S, 5, 60, S - 1])):
            b = _batch(inner.config, S=S, lens=lens)
            b["sample_ids"] = torch.arange(4 * i, 4 * i + 4, device="cuda", dtype=torch.int32)
            batches.append(_pack(b) if i == 1 else b)
        for _ in range(3):
            opt.zero_grad()
            inner.arena.window = 5
            eng.accumulate(model, batches)
            torch.cuda.synchronize()
        grads.append(inner.arena.grad.clone())
    assert torch.isfinite(grads[0]).all() and grads[0].abs().max() > 0
    torch.testing.assert_close(grads[0], grads[1], rtol=1e-5, atol=1e-5 * float(grads[1].abs().max()))
