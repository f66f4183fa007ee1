"""Where the host time of a short micro-batch goes: the C++ layer calls alone against the same calls under autograd.

Prints, for one 8-sample x 128-token BERT-large micro-batch, the host time to enqueue (a) 24 direct calls of
`layer_forward`, (b) 24 direct calls of `layer_backward`, (c) the model's forward through Python + autograd and
(d) its backward through the autograd engine.  (c) - (a) and (d) - (b) are what the Python / autograd layer adds."""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
from pytorch_distributed_training_amd.data.synthetic import fixed_batch  # noqa: E402
from pytorch_distributed_training_amd.engine import Engine  # noqa: E402
from pytorch_distributed_training_amd.models.bert import build_model  # noqa: E402
from pytorch_distributed_training_amd.ops import native  # noqa: E402
from pytorch_distributed_training_amd.optim import AdamW  # noqa: E402

eng = Engine(fp16=True, seed=0)
model = build_model("bert-large-cased")
opt = AdamW(params=model.parameters(), lr=1e-5)
model, opt = eng.prepare(model, opt)
model.train()
B, S = 8, 128
b = fixed_batch(B, S, eng.unwrap_model(model).config.vocab_size, eng.device, seed=1)
for _ in range(3):
    out = model(**b)
    eng.backward(out.loss)
    opt.step()
    opt.zero_grad()
torch.cuda.synchronize()

C = native()
layers = eng.unwrap_model(model).bert.encoder.layers()
cfg = layers[0].cfg
H, A = cfg.hidden_size, cfg.num_attention_heads
x = torch.randn(B * S, H, device=eng.device, dtype=torch.float16)
mask = torch.ones(B, S, dtype=torch.int32, device=eng.device)
kvl = torch.full((B,), S, dtype=torch.int32, device=eng.device)
state = torch.tensor([1, 0], dtype=torch.int64, device=eng.device)
n = 20


def direct():
    tf = tb = 0.0
    for _ in range(n):
        saved = []
        h = x
        t0 = time.perf_counter()
        for i, l in enumerate(layers):
            outs = C.layer_forward(h, mask, kvl, l._native.w, state, B, S, A, 0.1, 0.1, 1e-12, 1, i, None, None, None, None, None, None, True)
            saved.append((h, outs[1:]))
            h = outs[0]
        t1 = time.perf_counter()
        dy = h
        for i in reversed(range(len(layers))):
            l = layers[i]
            hin, sv = saved[i]
            dy = C.layer_backward(dy, hin, list(sv), mask, kvl, l._native.w, l._native.g, state, B, S, A, 0.1, 0.1, 1, i,
                                  True, None, None, None, None, None, None)
        t2 = time.perf_counter()
        tf += t1 - t0
        tb += t2 - t1
        torch.cuda.synchronize()
    return tf / n * 1e3, tb / n * 1e3


def through_autograd():
    tf = tb = 0.0
    for _ in range(n):
        t0 = time.perf_counter()
        out = model(**b)
        t1 = time.perf_counter()
        eng.backward(out.loss)
        t2 = time.perf_counter()
        tf += t1 - t0
        tb += t2 - t1
        torch.cuda.synchronize()
    return tf / n * 1e3, tb / n * 1e3


for label, fn in (("direct C++ layer calls (24 layers)", direct), ("model forward / autograd backward", through_autograd)):
    fn()
    f, bw = fn()
    print(f"{label}: forward {f:.2f} ms, backward {bw:.2f} ms host time per micro-batch", flush=True)
# the same direct calls with the weight-gradient side stream off: what the fork / join events cost the host
C.set_wgrad_side_stream(0)
f, bw = direct()
print(f"direct, weight gradients on the main stream: forward {f:.2f} ms, backward {bw:.2f} ms", flush=True)
# ... and with the K split of forward / dgrad GEMMs off (one launch and one allocation less per split GEMM)
C.set_gemm_split_k(False)
f, bw = direct()
print(f"direct, main stream, no K split: forward {f:.2f} ms, backward {bw:.2f} ms", flush=True)
