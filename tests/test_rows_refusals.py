"""Embedding table: calls that would lose something silently are refused."""
import pytest
import torch

from vectordb_amd import rows as R

import rows_reference as ref


def test_inputs_that_require_a_gradient():
    table = torch.zeros((4, 8), requires_grad=True)
    ids = torch.zeros((3,), dtype=torch.int64)
    grad = torch.zeros((3, 8), requires_grad=True)
    with pytest.raises(ValueError, match="table requires a gradient"):
        R.rows_lookup_device(table, ids)
    with pytest.raises(ValueError, match="grad_out requires a gradient"):
        R.rows_grad_device(grad, ids, 4)
    # without one to record: on to the next check
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        R.rows_lookup_device(table, ids)
    with pytest.raises(ValueError, match="GPU"):
        R.rows_lookup_device(table.detach(), ids)
    with pytest.raises(ValueError, match="GPU"):
        R.rows_grad_device(grad.detach(), ids, 4)


@pytest.mark.gpu
def test_a_trained_table(gpu):
    """What is refused, and the way that is documented instead: the lookup detached, its gradient called."""
    dev = torch.device("cuda", gpu)
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)
    weight = torch.nn.Parameter(torch.randn((50, 24), generator=gen, device=dev))
    ids = torch.randint(0, 50, (200,), generator=gen, device=dev)
    with pytest.raises(ValueError, match="table requires a gradient"):
        R.rows_lookup_device(weight, ids, 2.0)
    table = R.int4_encode_device(weight, 32)  # codes have no gradient: encoding takes any rows
    with pytest.raises(ValueError, match="queries requires a gradient"):
        table.distances_device(weight[:3])
    assert table.search_batch_device(weight[:3], 1)[0].shape == (3, 1)  # and so does a search
    y = R.rows_lookup_device(weight.detach(), ids, 2.0).requires_grad_()
    target = torch.randn((200, 24), generator=gen, device=dev)
    (y * target).sum().backward()
    weight.grad = R.rows_grad_device(y.grad, ids, 50, 2.0)
    want, mag, cnt = ref.grad(target.double().cpu().numpy(), ids.cpu().numpy(), 50, 2.0)
    # an f32 sum of cnt terms and a product: as many roundings, each of at most 2^-24 of the magnitudes' sum
    assert bool((abs(weight.grad.double().cpu().numpy() - want) <= (cnt[:, None] + 1) * 2.0 ** -24 * mag * 1.001 + 1e-45).all())
    with torch.no_grad():
        assert torch.equal(R.rows_lookup_device(weight, ids, 2.0), y.detach())


def test_a_stream_of_another_device():
    """Neither the kernels nor the outputs' memory would be on it."""
    class Stream:
        device, cuda_stream = torch.device("cuda", 1), 0x1234

    with pytest.raises(ValueError, match="a stream of cuda:1 for tensors on cuda:0"):
        R._enter(torch.device("cuda", 0), Stream())
