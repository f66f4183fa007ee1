"""Checkpoints of models with position options: nothing that a file should hold starts afresh without a word."""
import os

import pytest
import torch
from safetensors.torch import load_file, save_file

from pytorch_distributed_training_amd.checkpoint import (load_pretrained, load_state_dict_into, load_training_state, save_pretrained,
                                                         save_training_state)
from pytorch_distributed_training_amd.models.bert import build_model
from pytorch_distributed_training_amd.models.config import preset
from pytorch_distributed_training_amd.parallel.pp import build_stage

POSITION = dict(relative_attention_num_buckets=16, relative_attention_max_distance=40, qk_norm=True, rotary_dim=32)
TABLE = "bert.encoder.layer.1.attention.self.relative_attention_bias.weight"
NORM = "bert.encoder.layer.0.attention.self.query_norm.weight"


def _trained(**over):
    torch.manual_seed(1)
    model = build_model("bert-tiny-nodrop", **{**POSITION, **over})
    with torch.no_grad():
        for n, p in model.named_parameters():
            if "relative_attention_bias" in n or "_norm.weight" in n:
                p.normal_()
    return model


def _drop(path, *names):
    sd = load_file(path)
    save_file({k: v for k, v in sd.items() if k not in names}, path, metadata={"format": "pt"})


@pytest.mark.parametrize("name", [TABLE, NORM])
def test_a_file_that_lacks_trained_parameters_is_refused(tmp_path, name):
    save_pretrained(_trained(), str(tmp_path))
    load_pretrained(str(tmp_path))
    _drop(os.path.join(tmp_path, "model.safetensors"), name)
    with pytest.raises(KeyError, match=name):
        load_pretrained(str(tmp_path))
    with pytest.raises(KeyError, match=name):
        load_state_dict_into(_trained(), load_file(os.path.join(tmp_path, "model.safetensors")))


@pytest.mark.parametrize("name", [TABLE, NORM])
def test_a_resumed_run_does_not_start_parameters_afresh(tmp_path, name):
    path = save_training_state(str(tmp_path), _trained(), extra={"global_step": 3})
    load_training_state(str(tmp_path), _trained())
    _drop(os.path.join(os.path.dirname(path), "model.safetensors"), name)
    with pytest.raises(KeyError, match=name):
        load_training_state(str(tmp_path), _trained())


@pytest.mark.parametrize("change", [dict(rotary_dim=0), dict(rotary_dim=64), dict(rotary_base=500.0), dict(qk_norm_eps=1e-3),
                                    dict(relative_attention_max_distance=60), dict(qk_norm=False), dict(relative_attention_num_buckets=0)])
def test_a_resumed_run_keeps_its_position_options(tmp_path, change):
    save_training_state(str(tmp_path), _trained(), extra={"global_step": 3})
    with pytest.raises(ValueError, match="position options"):
        load_training_state(str(tmp_path), _trained(**change))


def test_options_off_do_not_count():
    a, b = preset("bert-tiny", relative_attention_max_distance=64, qk_norm_eps=1e-3, rotary_base=5.0), preset("bert-tiny")
    assert a.position_fields() == b.position_fields() == {}


def test_options_are_switched_on_over_a_plain_checkpoint(tmp_path):
    plain = build_model("bert-tiny-nodrop")
    save_pretrained(plain, str(tmp_path))
    model = load_pretrained(str(tmp_path), **POSITION)
    sd = model.state_dict()
    assert sd[TABLE].abs().max() == 0 and (sd[NORM] == 1).all()
    _drop(os.path.join(tmp_path, "model.safetensors"), "bert.encoder.layer.0.attention.self.query.weight")
    with pytest.raises(KeyError):
        load_pretrained(str(tmp_path), **POSITION)
    with pytest.raises(ValueError, match="rotary_dim"):
        load_pretrained(str(tmp_path), rotary_dim=24)


@pytest.mark.parametrize("name", [TABLE, NORM])
@pytest.mark.parametrize("told", [False, True])
def test_stages_of_a_state_that_lacks_some_layers_are_refused(name, told):
    cfg = preset("bert-tiny-nodrop", **POSITION)
    full = {k: v for k, v in _trained().state_dict().items() if k != name}
    with pytest.raises(KeyError, match=name):
        for stage in range(2):
            build_stage(cfg, stage, 2, full, **(dict(saved_cfg=cfg) if told else {}))
    plain = build_model("bert-tiny-nodrop").state_dict()
    if told:  # the configuration has the options, the state none of their parameters
        with pytest.raises(KeyError):
            build_stage(cfg, 0, 2, plain, saved_cfg=cfg)
        build_stage(cfg, 0, 2, plain, saved_cfg=preset("bert-tiny-nodrop"))


@pytest.mark.parametrize("change", [dict(rotary_dim=32), dict(qk_norm=True), dict(relative_attention_num_buckets=16)])
def test_models_with_position_options_are_not_handed_to_transformers(change):
    """transformers would build the plain architecture and compute something else (a rotation has no weights to be left over)."""
    from pytorch_distributed_training_amd.checkpoint import to_transformers

    with pytest.raises(ValueError, match="position options"):
        to_transformers(build_model("bert-tiny-nodrop", **change))
