"""The words of a mask: a bit a token, whatever type holds the truth values."""
import pytest
import torch

from helpers import pkg


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 100, 4099])
@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8, torch.int32, torch.float32])
def test_words(vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    mask = torch.randint(0, 4, (3, vocab), generator=g).to(dtype)   # truth is what is not 0
    words = pkg().dispatch.allowed_words(mask)
    assert words.shape == (3, (vocab + 31) // 32) and words.dtype == torch.int32
    bits = (words[:, :, None] >> torch.arange(32)) & 1
    assert torch.equal(bits.reshape(3, -1)[:, :vocab] != 0, mask != 0) and not bits.reshape(3, -1)[:, vocab:].any()


def test_refusals():
    with pytest.raises(pkg().Ab2Error):
        pkg().dispatch.allowed_words(torch.ones(5, dtype=torch.bool))
