"""The bucket form of the text encoder over more tokens than the window form's training pass takes, on the MI355X.
Tolerances as in test_bucket_encoder_gpu.py, whose longest sums have some 4000 terms too."""
import numpy as np
import pytest
import torch

from conftest import gpu_available
from gpu_util import rel_err, report
from gradtts_amd.text_encoder import TextEncoder
from gradtts_amd.params import synthetic_text_encoder_state_dict
from oracle import blocks

pytestmark = pytest.mark.gpu


def test_values_and_gradients_past_4096_tokens():
    if not gpu_available():
        pytest.skip("no HIP device")
    kw = dict(n_vocab=61, n_feats=80, n_channels=32, filter_channels=64, filter_channels_dp=32, n_heads=1, n_layers=1,
              kernel_size=3, n_buckets=16)
    sd = synthetic_text_encoder_state_dict(7, **kw)
    enc = TextEncoder(61, 80, 32, 64, 32, 1, 1, 3, 0.0, n_buckets=16, max_distance=64)
    enc.load_state_dict({k: torch.from_numpy(v) for k, v in sd.items()}, strict=True)
    enc.cuda().eval()
    T, lengths = 4163, torch.tensor([4163])
    tokens = torch.from_numpy(np.random.default_rng(7).integers(0, 61, size=(1, T)))
    mu, logw, _ = enc(tokens.cuda(), lengths.cuda())
    gen = torch.Generator().manual_seed(4)
    gmu, glw = torch.randn(mu.shape, generator=gen).double(), torch.randn(logw.shape, generator=gen).double()
    ((mu * gmu.float().cuda()).sum() + (logw * glw.float().cuda()).sum()).backward()
    p = {k: torch.as_tensor(v).double().requires_grad_() for k, v in sd.items()}
    rmu, rlw, _ = blocks.bucket_text_encoder(p, tokens, lengths, 1, 1, 64)
    ((rmu * gmu).sum() + (rlw * glw).sum()).backward()
    report("long bucket encoder mu_x", rel_err(mu.detach().cpu().numpy(), rmu.detach().numpy()), 2e-5)
    report("long bucket encoder logw", rel_err(logw.detach().cpu().numpy(), rlw.detach().numpy()), 2e-5)
    named = dict(enc.named_parameters())
    top = max(float(v.grad.abs().max()) for v in p.values())
    err = {k: float((named[k].grad.cpu().double() - v.grad).abs().max() / max(float(v.grad.abs().max()), 1e-3 * top))
           for k, v in p.items()}
    worst = max(err, key=err.get)
    report(f"long bucket encoder gradients (worst {worst})", err[worst], 1e-4)
    with torch.no_grad():
        again = enc(tokens.cuda(), lengths.cuda())
    report("long bucket encoder inference", rel_err(again[0].cpu().numpy(), rmu.detach().numpy()), 2e-5)
