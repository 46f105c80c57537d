"""Dropout from the counter-based generator: mask and values bit for bit against the oracle's hash."""
import numpy as np
import pytest
import torch

from oracle import fa2_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(x, p, seed, row0=0):
    rows, cols = x.reshape(-1, x.shape[-1]).shape
    keep = orc.dropout_keep(seed, np.arange(rows)[:, None] + row0, np.arange(cols)[None, :], 0, p)
    f = torch.tensor(1.0 / (1.0 - float(np.float32(p))), dtype=torch.float32)
    keep = torch.from_numpy(keep).view(x.shape).to(x.device)
    return torch.where(keep, x.float() * f.to(x.device), 0.0).to(x.dtype)


@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 64), (2, 3, 768), (510, 771), (2, 2, 2, 9), (1000, 1), (17,),
                                   (2500, 1032)])
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.999])
def test_values_and_gradient(fa, shape, t, p):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(t).to(DEV).requires_grad_(True)
    dy = torch.randn(*shape, generator=torch.Generator().manual_seed(2)).to(t).to(DEV)
    y = fa.dropout(x, p, seed=0xFFFFFFF1)
    (g,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(y, reference(x.detach(), p, 0xFFFFFFF1))
    assert torch.equal(g, reference(dy, p, 0xFFFFFFF1))


def test_layouts(fa):
    x = torch.randn(12, 64, device=DEV).half()
    ref = fa.dropout(x, 0.3, seed=9)
    wide = torch.cat([x, x], 1)
    assert torch.equal(fa.dropout(wide[:, :64], 0.3, seed=9), ref)
    assert torch.equal(fa.dropout(wide[:, 1:65], 0.3, seed=9), reference(wide[:, 1:65], 0.3, 9))
    assert torch.equal(fa.dropout(x.view(3, 4, 64).transpose(0, 1), 0.3, seed=9),
                       reference(x.view(3, 4, 64).transpose(0, 1).contiguous(), 0.3, 9))
    assert torch.equal(fa.dropout(x.t(), 0.3, seed=9), reference(x.t().contiguous(), 0.3, 9))
    one = x[:1].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(fa.dropout(one.expand(12, 64), 0.3, seed=9).float().sum(), one)
    f = reference(torch.ones(12, 64, device=DEV, dtype=torch.float16), 0.3, 9)
    assert torch.allclose(g.float(), f.float().sum(0, keepdim=True), rtol=2e-2)
    assert fa.dropout(x[:0], 0.3).shape == (0, 64) and fa.dropout(x[:, :0], 0.3).shape == (12, 0)
    assert fa.dropout(x, 0.0) is x


def test_masked_infinities_and_seeds(fa):
    x = torch.full((64, 64), float("inf"), device=DEV)
    x[::2] = float("nan")
    y = fa.dropout(x, 0.5, seed=4)
    keep = torch.from_numpy(orc.dropout_keep(4, np.arange(64)[:, None], np.arange(64)[None, :], 0, 0.5)).to(DEV)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    one = torch.ones(256, 256, device=DEV)
    a, b = fa.dropout(one, 0.25), fa.dropout(one, 0.25)
    assert not torch.equal(a, b)   # the module's counter moves on
    for m in (a, b):   # keep rate: 65536 draws of 0.75, six standard deviations
        assert abs((m > 0).double().mean().item() - 0.75) < 6 * (0.75 * 0.25 / 65536) ** 0.5


def test_more_elements_than_32_bits(fa):
    """A tensor of over 2^32 elements: its last rows."""
    rows, cols = (1 << 32) // 4096 + 3, 4096
    x = torch.ones(rows, cols, device=DEV, dtype=torch.float16)
    y = fa.dropout(x, 0.5, seed=77)
    assert torch.equal(y[-4:], reference(x[-4:], 0.5, 77, row0=rows - 4))
    assert torch.equal(y[:3], reference(x[:3], 0.5, 77))


def test_refusals(fa):
    x = torch.zeros(4, 8, device=DEV)
    for call in (lambda: fa.dropout(x, 1.0), lambda: fa.dropout(x, -0.1), lambda: fa.dropout(x.double(), 0.1),
                 lambda: fa.dropout(x[0, 0], 0.1), lambda: fa.dropout(x.cpu(), 0.1)):
        with pytest.raises(ValueError):
            call()


def test_probability_that_rounds_to_one_is_refused(fa):
    x, w = torch.zeros(4, 8, device=DEV), torch.ones(8, device=DEV)
    for call in (lambda: fa.dropout(x, 1 - 1e-9), lambda: fa.add_rms_norm(x, x, w, dropout_p=1 - 1e-9)):
        with pytest.raises(ValueError):
            call()
