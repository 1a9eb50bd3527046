"""The bucket form of the text encoder at widths and head sizes off every grid of its kernels, on the MI355X.
Tolerances as in test_bucket_encoder_gpu.py."""
import numpy as np
import pytest
import torch

from conftest import gpu_available
from gpu_util import rel_err, report
from gradtts_amd.params import synthetic_text_encoder_state_dict
from gradtts_amd.text_encoder import TextEncoder
from oracle import blocks

pytestmark = pytest.mark.gpu

# channels, FFN channels, predictor channels, features, heads, layers, kernel, lengths
CASES = [(35, 77, 33, 80, 5, 2, 3, [41, 1, 17]), (250, 131, 255, 7, 2, 1, 5, [33, 20]), (54, 1, 1, 128, 1, 2, 1, [64, 65, 3]),
         (255, 510, 200, 80, 255, 1, 3, [9]), (127, 254, 64, 1, 1, 1, 3, [130, 2])]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_values_and_gradients(case):
    if not gpu_available():
        pytest.skip("no HIP device")
    C, F, Fd, NF, H, L, K, lengths = case
    kw = dict(n_vocab=61, n_feats=NF, n_channels=C, filter_channels=F, filter_channels_dp=Fd, n_heads=H, n_layers=L,
              kernel_size=K, n_buckets=12)
    sd = synthetic_text_encoder_state_dict(5, **kw)
    enc = TextEncoder(61, NF, C, F, Fd, H, L, K, 0.0, n_buckets=12, max_distance=33)
    enc.load_state_dict({k: torch.from_numpy(v) for k, v in sd.items()}, strict=True)
    enc.cuda().eval()
    tokens = torch.from_numpy(np.random.default_rng(5).integers(0, 61, size=(len(lengths), max(lengths))))
    lengths = torch.tensor(lengths)
    mu, logw, _ = enc(tokens.cuda(), lengths.cuda())
    gen = torch.Generator().manual_seed(4)
    gmu, glw = torch.randn(mu.shape, generator=gen).double(), torch.randn(logw.shape, generator=gen).double()
    ((mu * gmu.float().cuda()).sum() + (logw * glw.float().cuda()).sum()).backward()
    p = {k: torch.as_tensor(v).double().requires_grad_() for k, v in sd.items()}
    rmu, rlw, _ = blocks.bucket_text_encoder(p, tokens, lengths, L, H, 33)
    ((rmu * gmu).sum() + (rlw * glw).sum()).backward()
    with torch.no_grad():
        again = enc(tokens.cuda(), lengths.cuda())
    for name, out in (("training pass", (mu, logw)), ("inference", again)):
        report(f"bucket encoder {name} mu_x {case}", rel_err(out[0].detach().cpu().numpy(), rmu.detach().numpy()), 2e-5)
        report(f"bucket encoder {name} logw {case}", rel_err(out[1].detach().cpu().numpy(), rlw.detach().numpy()), 2e-5)
    named = dict(enc.named_parameters())
    top = max(float(v.grad.abs().max()) for v in p.values())
    err = {k: float((named[k].grad.cpu().double() - v.grad).abs().max() / max(float(v.grad.abs().max()), 1e-3 * top))
           for k, v in p.items()}
    worst = max(err, key=err.get)
    report(f"bucket encoder gradients {case} (worst {worst})", err[worst], 1e-4)
