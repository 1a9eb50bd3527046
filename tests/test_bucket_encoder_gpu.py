"""The text encoder's bucket form (bucket attention joined by residual steps) on the MI355X, against its 64-bit
restatement (oracle.blocks.bucket_text_encoder) and torch's autograd through it.

Tolerances: a product over n channels in fp32 is off by about sqrt(n) 2^-24 of its norm, n at most 5 x 768: 4e-6. Some
three blocks' errors of that size stand in an output at full weight (the norms rescale, the stream adds): values 2e-5 of
the largest. A gradient passes both directions of every block: five times that, 1e-4 of the parameter's largest
gradient, or of a thousandth of the largest of all (the keys' bias has none: it shifts all of a row's scores).
"""
import numpy as np
import pytest
import torch

from conftest import gpu_available
from gpu_util import rel_err, report
from gradtts_amd import _lib
from gradtts_amd.params import synthetic_text_encoder_state_dict
from gradtts_amd.text_encoder import TextEncoder
from oracle import blocks
from oracle import text_encoder as ote

pytestmark = pytest.mark.gpu

# channels, heads, layers, kernel, buckets, max_distance, lengths
CASES = [(192, 2, 6, 3, 32, 128, [37, 21, 1]), (192, 2, 2, 3, 8, 9, [130, 97]), (160, 5, 2, 5, 16, 40, [33, 64, 50]),
         (128, 1, 2, 1, 4, 2, [40]), (48, 4, 2, 3, 10, 30, [29, 0, 17]), (256, 2, 1, 3, 128, 1024, [1]),
         (96, 4, 1, 3, 32, 128, [400, 333])]


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not gpu_available():
        pytest.skip("no HIP device")


def make(case, seed=3):
    C, H, L, K, nb, md, lengths = case
    kw = dict(n_vocab=61, n_feats=80, n_channels=C, filter_channels=4 * C, filter_channels_dp=96, n_heads=H, n_layers=L,
              kernel_size=K, n_buckets=nb)
    sd = synthetic_text_encoder_state_dict(seed, **kw)
    enc = TextEncoder(61, 80, C, 4 * C, 96, H, L, K, 0.1, n_buckets=nb, max_distance=md)
    enc.load_state_dict({k: torch.from_numpy(v) for k, v in sd.items()}, strict=True)
    rng = np.random.default_rng(seed)
    tokens = torch.from_numpy(rng.integers(0, 61, size=(len(lengths), max(lengths))))
    return enc.cuda().eval(), sd, tokens, torch.tensor(lengths)


@pytest.mark.parametrize("case", CASES, ids=str)
def test_values(case):
    enc, sd, tokens, lengths = make(case)
    p = {k: torch.as_tensor(v).double() for k, v in sd.items()}
    mu, logw, m = blocks.bucket_text_encoder(p, tokens, lengths, case[2], case[1], case[5])
    with torch.no_grad():
        got = enc(tokens.cuda(), lengths.cuda())
    taped = enc(tokens.cuda(), lengths.cuda())   # with gradients: the training pass, no dropout in eval mode
    for name, out in (("inference", got), ("training pass", taped)):
        report(f"bucket encoder {name} mu_x {case}", rel_err(out[0].detach().cpu().numpy(), mu.numpy()), 2e-5)
        report(f"bucket encoder {name} logw {case}", rel_err(out[1].detach().cpu().numpy(), logw.numpy()), 2e-5)
        assert torch.equal(out[2].cpu().double(), m)


@pytest.mark.parametrize("p_drop", [0.0, 0.1])
@pytest.mark.parametrize("case", CASES[:5], ids=str)
def test_gradients_of_every_parameter(case, p_drop):
    enc, sd, tokens, lengths = make(case)
    enc.train(p_drop > 0)
    enc.p_dropout = p_drop
    torch.manual_seed(3)
    seed = int(torch.randint(0, 2 ** 62, (1,)).item()) if p_drop else 0
    torch.manual_seed(3)
    mu, logw, _ = enc(tokens.cuda(), lengths.cuda())
    gen = torch.Generator().manual_seed(4)
    gmu, glw = torch.randn(mu.shape, generator=gen).double(), torch.randn(logw.shape, generator=gen).double()
    ((mu * gmu.float().cuda()).sum() + (logw * glw.float().cuda()).sum()).backward()
    p = {k: torch.as_tensor(v).double().requires_grad_() for k, v in sd.items()}
    drop = ote.Dropouts(seed, p_drop, 0.5) if p_drop else None
    rmu, rlw, _ = blocks.bucket_text_encoder(p, tokens, lengths, case[2], case[1], case[5], drop)
    ((rmu * gmu).sum() + (rlw * glw).sum()).backward()
    report(f"bucket encoder mu_x p={p_drop} {case}", rel_err(mu.detach().cpu().numpy(), rmu.detach().numpy()), 2e-5)
    named = dict(enc.named_parameters())
    assert set(named) == set(sd)
    top = max(float(v.grad.abs().max()) for v in p.values())
    err = {k: float((named[k].grad.cpu().double() - v.grad).abs().max() / max(float(v.grad.abs().max()), 1e-3 * top))
           for k, v in p.items()}
    worst = max(err, key=err.get)
    report(f"bucket encoder gradients p={p_drop} {case} (worst {worst})", err[worst], 1e-4)


def test_batch_entries_do_not_see_their_padding_or_each_other():
    case = CASES[0]
    enc, _, tokens, lengths = make(case)
    other = tokens.clone()
    for b, n in enumerate(lengths.tolist()):
        other[b, n:] = (other[b, n:] + 7) % 61
    with torch.no_grad():
        a, b = (enc(t.cuda(), lengths.cuda()) for t in (tokens, other))
        for x, y in zip(a, b):
            assert torch.equal(x, y)
        alone = enc(tokens[1:2, :21].cuda(), lengths[1:2].cuda())
    report("bucket encoder alone against batched", rel_err(alone[0].cpu().numpy(), a[0][1:2, :, :21].cpu().numpy()), 2e-5)


def test_training_repeats_and_follows_its_parameters():
    enc, _, tokens, lengths = make(CASES[2])
    enc.train()
    runs = []
    for _ in range(2):
        enc.zero_grad()
        torch.manual_seed(5)
        mu, logw, _ = enc(tokens.cuda(), lengths.cuda())
        (mu.square().sum() + logw.sum()).backward()
        runs.append([mu.detach().clone()] + [q.grad.clone() for q in enc.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    mu, logw, _ = enc(tokens.cuda(), lengths.cuda())
    with torch.no_grad():
        for q in enc.parameters():
            q -= 1e-3 * q.grad
    enc.eval()
    with torch.no_grad():
        stepped = enc(tokens.cuda(), lengths.cuda())[0]
    p = {k: v.detach().cpu().double() for k, v in enc.state_dict().items()}
    want = blocks.bucket_text_encoder(p, tokens, lengths, CASES[2][2], CASES[2][1], CASES[2][5])[0]
    report("bucket encoder after a step", rel_err(stepped.cpu().numpy(), want.numpy()), 2e-5)
    with pytest.raises(_lib.GradTTSError, match="no forward_train tape|parameters changed"):
        mu.sum().backward()


def test_whole_model_speaks_and_trains():
    from gradtts_amd.tts import GradTTS
    m = GradTTS(149, 1, 64, 192, 768, 256, 2, 2, 3, 0.1, None, 80, 64, 0.05, 20.0, 1000, n_buckets=32,
                max_distance=128).cuda()
    gen = torch.Generator().manual_seed(1)
    tokens, lengths = torch.randint(0, 149, (2, 31), generator=gen), torch.tensor([31, 20])
    mel, mel_lengths = torch.randn(2, 80, 96, generator=gen), torch.tensor([96, 72])
    m.train()
    losses = m.compute_loss(tokens.cuda(), lengths.cuda(), mel.cuda(), mel_lengths.cuda(), out_size=64)
    sum(losses).backward()
    assert all(torch.isfinite(q.grad).all() for q in m.encoder.parameters())
    assert float(m.encoder.encoder.attn_layers[0].table.grad.abs().max()) > 0
    m.eval()
    enc, dec, attn = m(tokens.cuda(), lengths.cuda(), n_timesteps=2)
    assert torch.isfinite(dec).all() and enc.shape == dec.shape and attn.shape[2] == 31
