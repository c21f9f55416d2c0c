"""The embedding's gradient where an id's places end and begin with the parts they are summed in (csrc/kernels/embedding.cu): 32 places of the sorted list a CTA, and 32 parts joined at
a time, so borders are at 32, 1024 and their multiples."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24


@pytest.mark.parametrize("before", [0, 1, 31, 32, 33, 1000, 1023])
@pytest.mark.parametrize("often", [1, 2, 31, 32, 33, 64, 65, 992, 1023, 1024, 1025, 1056, 2048, 2049, 33000])
@pytest.mark.parametrize("dt,hidden", [(torch.bfloat16, 40), (torch.float32, 9)])
def test_an_id_at_the_borders_of_parts(often, before, dt, hidden):
    """One id in ``often`` places behind ``before`` places of other ids, each of which comes once, and 40 places of further ones behind it."""
    from fuselink_b200.ops.embedding import lookup
    vocab = before + 60
    ids = torch.cat([torch.arange(before), torch.full((often,), before + 2), before + 5 + torch.arange(40)])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(often))].cuda()
    gen = torch.Generator(device="cuda").manual_seed(3)
    table = torch.randn(vocab, hidden, generator=gen, device="cuda").to(dt).requires_grad_(True)
    dout = torch.randn(len(ids), hidden, generator=gen, device="cuda").to(dt)
    got, = torch.autograd.grad(lookup(table, ids, 1.5), table, dout)
    again, = torch.autograd.grad(lookup(table, ids, 1.5), table, dout)
    assert torch.equal(got, again)
    want = torch.zeros(vocab, hidden, dtype=torch.float64, device="cuda").index_add(0, ids, dout.double())
    size = torch.zeros(vocab, hidden, dtype=torch.float64, device="cuda").index_add(0, ids, dout.double().abs())
    # a place goes through 32 sums of its part, 32 of its group of parts and one per group at most, each a half step of what there is; then the factor and the type's own rounding
    tol = 1.5 * size * (66 + often / 1024) * HALF + (1.5 * want).abs() * torch.finfo(dt).eps / 2 + torch.finfo(dt).tiny
    assert ((got.double() - 1.5 * want).abs() <= tol).all()
    assert (got[before] == 0).all() and (got[before + 50:] == 0).all()
