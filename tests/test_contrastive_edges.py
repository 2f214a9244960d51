"""The contrastive loss's operators where sizes, values and strides leave the ordinary range; tolerances as in test_contrastive.py."""
import pytest
import torch

from tests.test_contrastive import TYPES, bank_case


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [300.0, -300.0])
@pytest.mark.parametrize("S,V,ch", [(70, 333, 100), (33, 31, 24), (140, 65, 200)])
def test_scores_far_below_zero_with_a_list(gpu, S, V, ch, scale, dtype):
    """The zeros behind the last bank row must not count beside scores of -300, in the forms for lists too.  Rows on a grid of 1/128: products are
    exact, and so is their multiple by 300, so the order of the best entries is that of 64 bits."""
    gen = torch.Generator(device=gpu).manual_seed(3)
    u = torch.nn.functional.normalize(torch.randn(1, ch, generator=gen, device=gpu), dim=1)
    near = lambda n: torch.round(128 * torch.nn.functional.normalize(u + 0.02 * torch.randn(n, ch, generator=gen, device=gpu), dim=1)) / 128
    f, b = near(S).to(TYPES[dtype]), (near(V) * (-1.0 if scale > 0 else 1.0)).to(TYPES[dtype])
    for top in (1, 5, 16):
        bank_case(gpu, S, V, ch, TYPES[dtype], "none", top, scale=scale, features=f, bank=b)
    bank_case(gpu, S, V, ch, TYPES[dtype], "rows", 5, scale=scale, features=f, bank=b)
