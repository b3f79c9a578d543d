"""Every step of a sampler's rules is the f32 operation that it says: a quotient is rounded once, whatever the penalty."""
import pytest
import torch

from helpers import pkg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [4096, 4099])   # wide loads, single ones
@pytest.mark.parametrize("rho", [1.1, 1.3, 0.7, 3.0, 1e-30, 3e38, 1e-39])
def test_a_repeated_token_is_divided(vocab, rho):
    """torch divides and multiplies f32 with one rounding each; penalties of 0 subtract nothing."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    z = torch.randn(3, vocab, generator=g, device="cuda") * 4
    r = torch.full((3, 1), rho, device="cuda")
    rules = torch.cat([r, torch.zeros(3, 2, device="cuda")], dim=1)
    history = torch.arange(vocab, dtype=torch.int32, device="cuda").repeat(3, 1)
    got = pkg().dispatch.adjust_logits(z, history, None, rules)
    want = torch.where(z > 0, z / r, z * r)
    assert torch.equal(got, want), f"{int((got != want).sum())} of {want.numel()}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rho", [1.1, 3.0, 1e-30, 3e38, 1e-39])
def test_a_repeated_token_of_16_bits_is_divided(dtype, rho):
    """A product with the rounded reciprocal is off by 2^-23 of the quotient, then half a step of the type (below its normal numbers, of those); past its largest
    number it is infinite."""
    z = torch.randn(2, 2048, device="cuda").to(dtype)
    r = torch.full((2, 1), rho, device="cuda")
    got = pkg().dispatch.adjust_logits(z, torch.arange(2048, dtype=torch.int32, device="cuda").repeat(2, 1), None, torch.cat([r, torch.zeros(2, 2, device="cuda")], dim=1))
    zd, info = z.double(), torch.finfo(dtype)
    want = torch.where(zd > 0, zd / r.double(), zd * r.double())
    off = torch.clamp(want.abs() * (info.eps / 2 + 2.0 ** -23), min=info.eps * info.tiny / 2 * 1.001)
    inside = want.abs() < info.max * (1 - info.eps)
    assert ((got.double() - want).abs()[inside] <= off[inside]).all()
    assert torch.equal(got[want.abs() > info.max * (1 + info.eps)].double().abs(), torch.full_like(want[want.abs() > info.max * (1 + info.eps)], float("inf")))


def test_the_steps_in_their_order():
    g = torch.Generator(device="cuda").manual_seed(1)
    z, vocab = torch.randn(2, 1000, generator=g, device="cuda") * 4, 1000
    rules = torch.tensor([[1.3, 0.5, 0.25], [0.9, -0.5, 0.125]], device="cuda")   # whose sums with whole counts are exact
    history = torch.randint(0, vocab, (2, 3000), generator=g, device="cuda", dtype=torch.int32)
    count = torch.stack([torch.bincount(h.long(), minlength=vocab) for h in history]).float()
    ids = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:100] for _ in range(2)]).int()
    bias = torch.randn(2, 100, generator=g, device="cuda")
    rho, presence, frequency = (rules[:, i:i + 1] for i in range(3))
    want = torch.where(count > 0, torch.where(z > 0, z / rho, z * rho) - (presence + frequency * count), z)
    want = want.scatter(1, ids.long(), want.gather(1, ids.long()) + bias)
    assert torch.equal(pkg().dispatch.adjust_logits(z, history, None, rules, ids, bias), want)
