"""The example that runs the token operators together: packing on the CPU; on the
GPU a training run, and serving over the cache against the whole sequence at once."""

import pytest
import torch

from examples import image_tokens as E


def test_packed_documents():
    g = torch.Generator().manual_seed(1)
    pairs = [(torch.randn(n, 4, generator=g), torch.randn(n, 4, generator=g))
             for n in (1, 3, 2)]
    tokens, positions, documents, prefix, predicts, target = E.packed(pairs, torch.float32)
    assert tokens.shape == (1, 1 + 5 + 3, 5)
    assert positions[0].tolist() == [0, 0, 1, 2, 3, 4, 0, 1, 2]
    assert documents.tolist() == [[0, 1, 6, 9]] and prefix.tolist() == [[1, 3, 2]]
    assert predicts.tolist() == [True, False, False, True, True, True, False, True, True]
    assert target.shape == (6, 4)
    assert torch.equal(tokens[0, 4, :4], pairs[1][0][0]) and tokens[0, 4, 4] == 1


def test_no_cuda_is_said(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    with pytest.raises(SystemExit, match="needs a CUDA device"):
        E.main([])
    model = E.ImageTokens(4, dim=32, heads=2, key_heads=1, width=16, layers=1, rows=16)
    with pytest.raises(RuntimeError, match="expects CUDA tensors"):
        model(torch.zeros(1, 3, 5), torch.arange(3)[None])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_training_lowers_the_loss(cuda, dtype):
    torch.manual_seed(0)
    g = torch.Generator(device=cuda).manual_seed(0)
    model = E.ImageTokens(16).to(cuda, E.DTYPES[dtype])
    losses = E.train(model, 60, E.DTYPES[dtype], 4, g)
    # predicting zero leaves the noise's mean square, a quarter
    assert sum(losses[-5:]) / 5 < 0.75 * sum(losses[:3]) / 3
    assert model.mix[0].bias.grad.abs().sum() > 0
    assert model.mix[0].q_weight.grad.abs().sum() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("B, n", [(1, 1), (3, 7), (2, 49)])
def test_serving_agrees_with_the_whole_sequence(cuda, B, n):
    """Each served patch is what the model gives for the sequence so far in one
    call.  fp32: an fp32 sum of a few hundred terms is good to 1e-6 of its size,
    six such products and two softmaxes to 1e-4 of the outputs near one."""
    torch.manual_seed(1)
    g = torch.Generator(device=cuda).manual_seed(1)
    model = E.ImageTokens(16).to(cuda)
    for m in model.mix:
        torch.nn.init.normal_(m.bias)
    noisy = torch.randn(B, n, 16, generator=g, device=cuda)
    served = E.denoise(model, noisy)
    assert served.shape == (B, n, 16)
    tokens = torch.cat([E.marked(noisy, False), E.marked(served[:, :-1], True)], 1)
    at = torch.arange(2 * n - 1, device=cuda).expand(B, -1)
    with torch.no_grad():
        whole = model(tokens, at, prefix=n)[:, n - 1:] + noisy
    torch.testing.assert_close(served, whole, rtol=1e-4, atol=1e-4)
