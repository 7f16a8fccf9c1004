"""The token-hash text encoder on the GPU is what it is on the CPU: an indexing of its table by any ids that torch takes, an error for others,
in the type the module has."""
import pytest
import torch


class _OnGpu(torch.Tensor):
    """Passes for a GPU tensor; what launches a kernel for it without one fails."""
    is_cuda = True


def _pair(dtype=torch.float32):
    from diffuser.libero.lb_train_utils import HashTextEncoder
    enc = HashTextEncoder(dim=16, vocab=50, max_len=8).to(dtype)
    want = HashTextEncoder(dim=16, vocab=50, max_len=8).to(dtype)
    enc.table = enc.table.as_subclass(_OnGpu)
    return enc, want


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_ids_index_the_table(dtype):
    enc, want = _pair(dtype)
    ids = torch.tensor([[3, 49, -1], [-50, 0, 7]])           # negative ones count from the end
    got = enc(ids.as_subclass(_OnGpu)).last_hidden_state
    assert got.dtype == dtype and torch.equal(got.as_subclass(torch.Tensor), want(ids).last_hidden_state)
    assert torch.equal(want(ids).last_hidden_state, (want.table[ids % 50] + want.pos[None, :3]))


@pytest.mark.parametrize("bad", [50, -51, 2 ** 40])
def test_ids_outside_the_table_are_an_error(bad):
    enc, want = _pair()
    ids = torch.tensor([[3, bad]])
    for e, i in ((want, ids), (enc, ids.as_subclass(_OnGpu))):
        with pytest.raises(IndexError):
            e(i)


def test_other_id_types():
    enc, want = _pair()
    ids = torch.tensor([[3, 4], [5, 6]])
    got = enc(ids.int().as_subclass(_OnGpu)).last_hidden_state
    assert torch.equal(got.as_subclass(torch.Tensor), want(ids).last_hidden_state)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16])
def test_the_same_values_on_the_gpu(dtype):
    from diffuser.libero.lb_train_utils import HashTextEncoder
    enc = HashTextEncoder(dim=16, vocab=50, max_len=8).to(dtype)
    ids = torch.tensor([[3, 49, -1], [-50, 0, 7]])
    want = enc(ids).last_hidden_state
    enc = enc.cuda()
    for i in (ids.cuda(), ids.int().cuda(), ids):
        assert torch.equal(enc(i).last_hidden_state.cpu(), want)
