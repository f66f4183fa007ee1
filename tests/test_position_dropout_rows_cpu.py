"""Dropout rows of models whose position table is longer than 512 tokens: a sample's rows are its own."""
import pytest
import torch

from pytorch_distributed_training_amd.models.bert import build_model
from pytorch_distributed_training_amd.models.config import preset
from pytorch_distributed_training_amd.ops import fused
from pytorch_distributed_training_amd.ops.arena import ParamArena


def _packed_rows(monkeypatch, model, lens, S, sample_ids):
    """rowmap of a packed batch, as the encoder stack receives it."""
    seen = {}
    monkeypatch.setattr(fused, "embeddings_forward_packed", lambda emb, ids, types, pos, rowmap, ie: torch.zeros(len(ids), 8))
    monkeypatch.setattr(fused, "encoder_stack_forward", lambda layers, x, mask: seen.setdefault("mask", mask) and x)
    mask = torch.arange(S)[None] < torch.tensor(lens)[:, None]
    cu = torch.nn.functional.pad(mask.sum(1).cumsum(0), (1, 0))
    model._forward_unpadded(torch.ones(len(lens), S, dtype=torch.int64), None, None, sample_ids, cu,
                            mask.reshape(-1).nonzero().flatten(), run_head=False)
    return seen["mask"].rowmap.to(torch.int64) & 0xFFFFFFFF, mask


@pytest.mark.parametrize("positions,model_type", [(128, "bert"), (512, "bert"), (513, "bert"), (1024, "bert"), (1500, "bert"), (514, "roberta"), (1026, "roberta")])
@pytest.mark.parametrize("with_ids", [False, True])
def test_packed_rows_belong_to_one_sample(monkeypatch, positions, model_type, with_ids):
    name = "bert-tiny" if model_type == "bert" else "roberta-tiny"
    model = build_model(name, max_position_embeddings=positions, rotary_dim=32)
    S = positions if model_type == "bert" else positions - 2
    ids = torch.tensor([4, 3, 5], dtype=torch.int32) if with_ids else None
    rows, mask = _packed_rows(monkeypatch, model, [S, S, S // 2], S, ids)
    assert len(rows.unique()) == len(rows)
    # padded rows of the same batch: the kernels form id * 512 + position from the ids that begin_forward() hands them
    arena = ParamArena(model, torch.device("cpu"))
    runtime = fused.NativeRuntime(arena)
    runtime.sample_blocks = model.config.dropout_blocks
    key = runtime.begin_forward(ids if with_ids else torch.arange(3))
    padded = key.sample_ids.to(torch.int64)[:, None] * 512 + torch.arange(S)
    assert torch.equal(rows, padded[mask])


def test_rows_of_up_to_512_positions_are_as_before(monkeypatch):
    model = build_model("bert-tiny", max_position_embeddings=512)
    rows, mask = _packed_rows(monkeypatch, model, [512, 7], 512, torch.tensor([9, 2]))
    assert torch.equal(rows, (torch.tensor([9, 2])[:, None] * 512 + torch.arange(512))[mask])
    assert {preset(n).dropout_blocks for n in ("bert-large-cased", "roberta-large", "bert-tiny", "roberta-tiny")} == {1}


def test_sequences_behind_the_last_position_are_refused():
    model = build_model("roberta-tiny", max_position_embeddings=514, rotary_dim=32)  # 512 tokens
    with pytest.raises(ValueError, match="positions allow"):
        fused.encoder_stack_forward(model.base_model.encoder.layers(), torch.zeros(1, 513, 128), type("M", (), {"seq": 513}))
