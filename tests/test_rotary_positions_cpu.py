"""rotary_embed's refusal of one position for all tokens, with sections: by name, as without them."""
import pytest
import torch

from cache_dit_amd import _native, rotary


@pytest.mark.parametrize("ends", [[], [16, 32]])
def test_one_position(monkeypatch, ends):

  class Host:

    def rotary(self, *args):
      return None

  monkeypatch.setattr(_native, "host", lambda: Host())
  with pytest.raises(ValueError, match="rotary_embed: positions"):
    rotary._rotary_general(torch.zeros(3, 2, 64), None, torch.tensor(5), torch.ones(32, dtype=torch.float64), None, None, None, None, 0, ends, 1.0, 1e-6)
