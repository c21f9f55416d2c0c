"""Embedding lookup and its gradient (csrc/kernels/embedding.cu) against the same in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16, torch.float32]


def _table(vocab, hidden, dt, seed=1):
    return torch.randn(vocab, hidden, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dt)


def _ids(n, vocab, seed=2, dtype=torch.int64, often=0.0):
    """Tokens in no order, a part of them the same one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    return torch.where(torch.rand(n, generator=g, device="cuda") < often, vocab // 3, ids).to(dtype)


def _check_grad(got, ids, dout, vocab, scale):
    """Sums of n values of one sign pattern are off by at most n half steps of fp32 of the sum of magnitudes, whatever their order; the factor adds
    one half step, and the table's type its own."""
    ids, x = ids.reshape(-1).long(), dout.reshape(-1, dout.shape[-1]).double()
    ids = torch.where(ids < 0, ids + vocab, ids)
    zero = torch.zeros(vocab, x.shape[1], dtype=torch.float64, device="cuda")
    want, size = zero.index_add(0, ids, x) * scale, zero.index_add(0, ids, x.abs()) * abs(scale)
    n = torch.bincount(ids, minlength=vocab).double()[:, None]
    tol = (n + 2) * 2.0 ** -24 * size + torch.finfo(got.dtype).eps / 2 * want.abs() + torch.finfo(got.dtype).smallest_normal
    assert ((got.double() - want).abs() <= tol).all()
    assert (got[n[:, 0] == 0] == 0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("n,vocab,hidden", [(1, 1, 1), (3, 5, 8), (16, 512, 128), (33, 1000, 7), (100, 63, 96), (257, 513, 1601), (1000, 1025, 4096), (5, 130, 5120), (2048, 64, 24)])
def test_lookup_and_gradient(n, vocab, hidden, dt):
    from fuselink_b200.ops.embedding import lookup
    table, ids = _table(vocab, hidden, dt).requires_grad_(True), _ids(n, vocab)
    scale = 1.5 * hidden ** 0.5
    out = lookup(table, ids, scale)
    assert torch.equal(out, (table.detach().float()[ids] * scale).to(dt)) and out.shape == (n, hidden)
    dout = torch.randn(n, hidden, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(dt)
    got, = torch.autograd.grad(out, table, dout)
    _check_grad(got, ids, dout, vocab, scale)


# an id in 1 to 32 places is one warp's, up to 1024 a CTA's, more are cut into parts of 1024 places
@pytest.mark.parametrize("often", [0.0, 0.01, 0.3, 0.97, 1.0])
@pytest.mark.parametrize("n", [1024, 1025, 2048, 5003, 40000])
@pytest.mark.parametrize("dt,hidden", [(torch.float32, 36), (torch.bfloat16, 264), (torch.float16, 5)])
def test_tokens_that_come_often(n, often, dt, hidden):
    from fuselink_b200.ops.embedding import lookup
    vocab = 700
    table, ids = _table(vocab, hidden, dt).requires_grad_(True), _ids(n, vocab, often=often)
    dout = torch.randn(n, hidden, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(dt)
    got, = torch.autograd.grad(lookup(table, ids), table, dout)
    _check_grad(got, ids, dout, vocab, 1.0)
    again, = torch.autograd.grad(lookup(table, ids), table, dout)
    assert torch.equal(got, again)                                    # the order of the sums is the tokens'


def test_two_tokens_of_many_places_in_one_part():
    """Ids that begin and end within the same part of the sorted list, behind one another."""
    from fuselink_b200.ops.embedding import lookup
    ids = torch.cat([torch.full((n,), v, device="cuda") for v, n in enumerate((1500, 1, 0, 3000, 40, 1024, 1025, 2047, 5000, 1, 1))])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")]
    table, dout = _table(11, 40, torch.float32).requires_grad_(True), torch.randn(len(ids), 40, device="cuda")
    got, = torch.autograd.grad(lookup(table, ids, 0.5), table, dout)
    _check_grad(got, ids, dout, 11, 0.5)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_shapes_types_strides_and_offsets(dtype):
    from fuselink_b200.ops.embedding import lookup
    wide = _table(300, 72, torch.bfloat16)
    table = wide[:, 3:67].requires_grad_(True)                        # rows of another distance, none at a multiple of 16 bytes
    ids = _ids(84, 300, dtype=dtype).view(7, 12).t()                  # [12, 7], not contiguous
    ids = torch.where(ids % 5 == 0, ids - 300, ids)                   # some counted from the end
    out = lookup(table, ids, 3.0)
    assert out.shape == (12, 7, 64) and torch.equal(out, (table.detach().float()[ids.long()] * 3).to(torch.bfloat16))
    dout = torch.randn(64, 12, 7, device="cuda").to(torch.bfloat16).permute(1, 2, 0)
    _check_grad(torch.autograd.grad(out, table, dout)[0], ids, dout.contiguous(), 300, 3.0)
    one = torch.tensor(5, dtype=dtype, device="cuda")
    assert torch.equal(lookup(table, one), table.detach()[5])
    same = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(12, 7, 64)                  # a gradient that is one value everywhere
    _check_grad(torch.autograd.grad(lookup(table, ids), table, same)[0], ids, same, 300, 1.0)
    none = lookup(table, ids[:0])
    assert none.shape == (0, 7, 64) and (torch.autograd.grad(none, table, none.detach())[0] == 0).all()


def test_a_token_outside_the_vocabulary():
    from fuselink_b200.ops.embedding import lookup
    word = torch.zeros(1, dtype=torch.int32).pin_memory()
    table = _table(10, 16, torch.float32).requires_grad_(True)
    ids = torch.tensor([3, -10, 9], device="cuda")
    lookup(table, ids, status=word.data_ptr())
    torch.cuda.synchronize()
    assert int(word) == 0
    ids = torch.tensor([3, 10, -11, 2 ** 40, -2 ** 40, 3], device="cuda")
    out = lookup(table, ids, status=word.data_ptr())
    got, = torch.autograd.grad(out, table, torch.ones_like(out))
    torch.cuda.synchronize()
    assert int(word) == 1
    assert (out[1:5] == 0).all() and torch.equal(out[0], table[3]) and got[3].eq(2).all() and got.sum() == 32


def test_captured_and_on_another_stream():
    from fuselink_b200.ops.embedding import lookup
    table, ids, dout = _table(500, 64, torch.bfloat16), _ids(300, 500, often=0.2), torch.randn(300, 64, device="cuda").to(torch.bfloat16)

    def both(t):
        leaf = t.detach().requires_grad_(True)                        # a leaf of the stream's own
        return torch.autograd.grad(lookup(leaf, ids, 2.0), leaf, dout)[0]

    want = both(table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(table)
        other = both(table)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(table)
    for seed in (11, 12):
        ids.copy_(_ids(300, 500, seed=seed, often=0.3))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, both(table))


def test_differences_of_the_loss():
    """The derivative along a direction against the difference of two losses: both are linear in the table, so only roundings part them."""
    from fuselink_b200.ops.embedding import lookup
    table, ids = _table(50, 16, torch.float32).requires_grad_(True), _ids(40, 50)
    c, d = torch.randn(40, 16, device="cuda"), torch.randn(50, 16, device="cuda")
    got = (torch.autograd.grad(lookup(table, ids, 2.0), table, c)[0] * d).double().sum()
    f = lambda t: (lookup(t, ids, 2.0).double() * c.double()).sum()  # noqa: E731
    want = (f(table.detach() + d) - f(table.detach() - d)) / 2
    # each of 640 products of values around 2 has a handful of half steps of fp32 in it
    assert abs(got - want) <= 640 * 16 * 2.0 ** -24 * 8


def test_what_is_refused():
    from fuselink_b200.ops.embedding import lookup
    table, ids = _table(10, 16, torch.float32), _ids(4, 10)
    for bad, args in ((RuntimeError, (table, ids.float())), (RuntimeError, (table, ids.cpu())), (ValueError, (table[0], ids)), (ValueError, (table[:0], ids)),
                      (RuntimeError, (table.double(), ids)), (RuntimeError, (table.t(), ids)), (RuntimeError, (table[:1].expand(10, 16), ids))):
        with pytest.raises(bad):
            lookup(*args)
    leaf = table.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiated"):
        torch.autograd.grad(lookup(leaf, ids).square().sum(), leaf, create_graph=True)
