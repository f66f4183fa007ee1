"""What layers with position options keep for their backward pass, against what the micro-batch size counts on."""
import gc

import pytest
import torch

from pytorch_distributed_training_amd.config import TrainConfig
from pytorch_distributed_training_amd.models.config import preset

OPTIONS = [dict(), dict(relative_attention_num_buckets=32), dict(rotary_dim=64), dict(relative_attention_num_buckets=32, qk_norm=True, rotary_dim=64)]


@pytest.mark.parametrize("option", OPTIONS)
@pytest.mark.parametrize("max_length,extra", [(128, 0), (512, 3)])
def test_micro_batches_count_what_the_options_keep(option, max_length, extra):
    cfg = TrainConfig(max_length=max_length)
    arch = preset("bert-large-cased", **option)
    per = 34 + (4 if arch.qk_norm or arch.rotary_dim else 0) + (extra if option else 0)
    free = 40 << 30
    assert cfg.micro_batch_cap(torch.device("cuda"), arch, free_bytes=free) == (free // 2) // (per * 24 * 1024) // max_length


@pytest.mark.gpu
@pytest.mark.parametrize("option", OPTIONS[1:])
@pytest.mark.parametrize("S", [128, 400])
def test_layers_keep_what_is_counted(option, S):
    from pytorch_distributed_training_amd.models.bert import MaskInfo, build_model
    from pytorch_distributed_training_amd.ops import fused
    from pytorch_distributed_training_amd.ops.arena import ParamArena

    B, L = 16, 4
    kept = []
    requested = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]  # (without the allocator's rounding to blocks)
    for over in (dict(), option):
        model = build_model("bert-tiny", max_position_embeddings=512, num_hidden_layers=L, **over).cuda()
        model.enable_native(ParamArena(model, torch.device("cuda"), torch.float16))
        model.train()
        H = model.config.hidden_size
        x = torch.randn(B, S, H, device="cuda").half().requires_grad_()
        mask = MaskInfo(None, B, S, x.device)
        model.runtime.begin_forward(None)
        for _ in range(2):  # (the first pass brings workspaces that stay)
            gc.collect()  # (models are cycles of references: those of earlier passes go now)
            before = requested()
            y = fused.encoder_stack_forward(model.bert.encoder.layers(), x, mask)
            kept.append((requested() - before) / (B * S * H * L))
            del y
    arch = preset("bert-tiny", **option)
    more = kept[3] - kept[1]
    counted = arch.saved_bytes(S) - 34
    assert counted - 1.1 <= more <= counted, (more, counted)
