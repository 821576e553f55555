"""lora_add's general path without a GPU: what is not laid out as the launcher takes it reaches the launcher laid out so, whatever the
form of ids. The launcher's stand-in has its conditions and computes."""
import pytest
import torch

from cache_dit_amd import _native, adapters
from oracle import block_oracle as bo

BF16 = torch.bfloat16


class Host:
  """The extension's conditions for a launch, and the oracle's result."""
  launches = 0

  def lora_add(self, base, x, down, up, ids, scale, rank, x_scale, epilogue):

    def rows(t):
      return t.stride(1) == 1 and t.shape[1] <= t.stride(0) < 1 << 24 if t.dim() == 2 else t.is_contiguous()

    if not (x.dim() == base.dim() and rows(x) and rows(base) and down.is_contiguous() and up.is_contiguous() and up.data_ptr() % 16 == 0
            and ids.dtype in (torch.int32, torch.int64) and ids.is_contiguous() and ids.dim() < x.dim()
            and ids.shape == x.shape[:ids.dim()]):
      return None
    for t, dtype in ((scale, torch.float32), (rank, torch.int32), (x_scale, torch.float32)):
      if t is not None and not (t.dtype == dtype and t.is_contiguous()):
        return None
    self.launches += 1
    count = base.shape[:-1].numel()
    each = ids.reshape(-1).repeat_interleave(count // ids.numel())
    out, _ = bo.lora(base.reshape(count, -1), x.reshape(count, -1), down, up, each, scale, rank, x_scale)
    return 0, out.to(BF16).view(base.shape)


@pytest.fixture
def host(monkeypatch):
  host = Host()
  monkeypatch.setattr(_native, "host", lambda: host)
  return host


def data(B, S, N=24, K=40):
  g = torch.Generator().manual_seed(0)
  return (torch.randn(B, S, N, generator=g).to(BF16), torch.randn(B, S, K, generator=g).to(BF16),
          torch.randn(2, 16, K, generator=g).to(BF16), torch.randn(2, N, 16, generator=g).to(BF16))


IDS = [torch.tensor(1), torch.tensor([1, 0, 1]), torch.tensor([[1], [0], [1]]).expand(3, 7), torch.tensor(0, dtype=torch.int16),
       torch.tensor([1, 0, -1], dtype=torch.int8)]


@pytest.mark.parametrize("ids", IDS)
@pytest.mark.parametrize("form", ["slice", "double scale", "transposed base"])
def test_any_ids_with_any_layout(host, ids, form):
  base, x, down, up = data(3, 7)
  scale, want_scale = torch.tensor([0.5, 2.0]), torch.tensor([0.5, 2.0])
  each = ids.long().reshape(-1).repeat_interleave(21 // ids.numel())
  if form == "slice":
    x, base = torch.cat((x, x), 1)[:, :7], torch.cat((base, base), 1)[:, :7]
  elif form == "double scale":
    scale = scale.double()
  else:
    base = base.transpose(0, 1).contiguous().transpose(0, 1)
  got = adapters._lora_add(base, x, down, up, ids, scale, None, None)
  want, _ = bo.lora(base.reshape(21, -1), x.reshape(21, -1), down, up, each, want_scale)
  assert got.shape == base.shape and torch.equal(got.view(21, -1), want.to(BF16)) and host.launches == 1


def test_one_request(host):
  base, x, down, up = data(1, 5)
  want, _ = bo.lora(base[0], x[0], down, up, torch.ones(5, dtype=torch.long))
  for ids in (torch.tensor(1), torch.tensor([1]), torch.tensor([1], dtype=torch.int16)):
    got = adapters._lora_add(base, torch.cat((x, x), 2)[..., :40], down, up, ids, None, None, None)
    assert torch.equal(got[0], want.to(BF16))
  got = adapters._lora_add(base[0, 0], x[0, 0], down, up, torch.tensor(1, dtype=torch.int8), None, None, None)
  assert got.shape == (24, ) and torch.equal(got, want[0].to(BF16))
  got = adapters._lora_add(base[0], torch.cat((x, x), 2)[0, :, ::2], down, up, torch.tensor(1, dtype=torch.int8), None, None, None)
  assert got.shape == (5, 24) and host.launches == 5


def test_ids_keep_their_rows_together(host, monkeypatch):
  """A request's rows reach the launcher as one, not as ids row by row."""
  seen = []
  plain = host.lora_add
  monkeypatch.setattr(host, "lora_add", lambda *a: (seen.append(a[4].numel()), plain(*a))[1])
  base, x, down, up = data(3, 7)
  adapters._lora_add(base, torch.cat((x, x), 1)[:, :7], down, up, torch.tensor([1, 0, 1]), None, None, None)
  assert seen[-1] == 3


def test_what_the_launcher_does_not_take_has_a_name(host, monkeypatch):
  monkeypatch.setattr(host, "lora_add", lambda *a: None)
  base, x, down, up = data(3, 7)
  with pytest.raises(RuntimeError, match="cdit::lora_add: .*not taken"):
    adapters._lora_add(base, x, down, up, torch.tensor(1), None, None, None)
