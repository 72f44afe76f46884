"""What the cross attention takes as text lengths, checked before any device work."""
import pytest
import torch

from icsa_hip import wan
from icsa_hip.hip_host import IcsaArgumentError

pytestmark = pytest.mark.cpu


@pytest.mark.parametrize("lens", [[1.5], torch.tensor([2.0]), torch.tensor([True]), [True]])
def test_text_lengths_are_whole_numbers(lens):
    ca = wan.WanT2VCrossAttention(256, 2)
    with pytest.raises(IcsaArgumentError, match="whole numbers"):
        ca(torch.randn(1, 4, 256), torch.randn(1, 6, 256), lens)


@pytest.mark.parametrize("lens", [[1, 2], torch.tensor([[3]]), torch.tensor(3)])
def test_one_length_a_batch_row(lens):
    ca = wan.WanT2VCrossAttention(256, 2)
    with pytest.raises(IcsaArgumentError, match="one length"):
        ca(torch.randn(1, 4, 256), torch.randn(1, 6, 256), lens)
