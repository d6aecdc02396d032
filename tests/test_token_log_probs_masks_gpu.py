"""Token log probabilities of rows that are masked in two ways at once, with the type's lowest number and with -inf, and of logits beyond 2^16: rows that begin on and off 16-byte boundaries, in each form of
the launch.  What a result may be off by does not grow with the masked values."""
import numpy as np
import pytest
import torch

from tests.util import NAME

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda d: NAME[d])
# few rows are dealt over workgroups of 256 threads, some hundred have workgroups of 512, many of 256
ROWS = pytest.mark.parametrize("rows", [3, 300, 700])
VOCAB = 9001


def _rows(kinds, rows, dtype, shift):
    """[rows, VOCAB] that begin `shift` values behind a 16-byte boundary, the kinds in turn."""
    flat = torch.zeros(rows * VOCAB + 16, dtype=dtype, device="cuda")
    x = flat[shift:shift + rows * VOCAB].view(rows, VOCAB)
    table = torch.stack([k.to(dtype) for k in kinds]).cuda()
    x.copy_(table[torch.arange(rows, device="cuda") % len(kinds)])
    return x


def _check(x, size, top=4):
    """Against float64, with `size` the largest logit that has a weight: 2 ** -24 for each of the sums' additions (VOCAB / 256 of a lane and the tree's), for the steps from logits of that size to
    their logarithm, and for the results' own."""
    from metalhlo_amd import kernels
    tokens = (torch.arange(x.shape[0], device="cuda") * 131 % VOCAB).int()
    log_p, entropy, top_p, top_id = (t.cpu().numpy() for t in kernels.token_log_probs(x, tokens, top=top))
    d = x.double().cpu()
    want = torch.log_softmax(d, 1)
    p = want.exp()
    want_entropy = -torch.where(p > 0, p * want, 0.0).sum(1).numpy()
    order = torch.sort(d, dim=1, descending=True, stable=True).indices[:, :top]
    step = 2.0 ** -24
    assert (top_id == order.numpy()).all()
    for got, index in ((log_p[:, None], tokens.cpu().long()[:, None]), (top_p, order)):
        w = want.gather(1, index).numpy()
        far = d.gather(1, index).abs().numpy()
        with np.errstate(invalid="ignore"):
            ok = (got == w) | (np.abs(got - w) <= step * (VOCAB / 256 + 64 + 8 * size + 8 * np.where(far > size, far, 0.0) + 8 * np.abs(w)))
        assert ok.all(), (np.argwhere(~ok)[:4], got[~ok][:4], w[~ok][:4])
    # (a weight of exponent -d is off by (4 + 2 d) 2 ** -24 and counts d times; d up to 40 where it counts at all)
    assert (np.abs(entropy - want_entropy) <= step * ((VOCAB / 256 + 64) * (1 + want_entropy + 8) + 84 * 50 + 8 * size)).all(), (entropy[:6], want_entropy[:6])


@TYPES
@ROWS
@pytest.mark.parametrize("shift", [0, 1, 3, 7])
def test_lowest_numbers_and_infinities_in_one_row(rows, shift, dtype):
    g = torch.Generator().manual_seed(7)
    low, inf = torch.finfo(dtype).min, float("inf")
    normal = torch.randn(VOCAB, generator=g).to(dtype).float() * 3
    i = torch.arange(VOCAB)
    begun = torch.where(i < 7, low, -inf)                     # the first values as one mask writes them, all the others as another
    kinds = [torch.where((i >= 5000) & (i < 5100), normal, begun),
             torch.where(i == 8999, normal, begun),
             torch.where(i < 4500, begun, normal),
             torch.where(torch.rand(VOCAB, generator=g) < 0.1, normal, torch.where(torch.rand(VOCAB, generator=g) < 0.5, low, -inf))]
    kinds += [torch.where((i // 1024) % 2 == 1, kinds[3], begun)]
    _check(_rows(kinds, rows, dtype, shift), 20.0)


@TYPES
@ROWS
@pytest.mark.parametrize("shift", [0, 1, 3, 7])
def test_lowest_numbers_alone_have_the_probability(rows, shift, dtype):
    """Of a row that holds the type's lowest number and -inf the former are equally likely."""
    low, inf = torch.finfo(dtype).min, float("inf")
    i = torch.arange(VOCAB)
    kinds = [torch.where(i < n, low, -inf) for n in (1, 7, 300, 5000)] + [torch.where(i >= VOCAB - 3, low, -inf), torch.where((i < 2) | (i == 2100), low, -inf)]
    x = _rows(kinds, rows, dtype, shift)
    from metalhlo_amd import kernels
    count = (x > -inf).sum(1)
    log_p, entropy, top_p, top_id = kernels.token_log_probs(x, (x > -inf).int().argmax(1), top=1)
    want = -count.double().log()
    # (equal logits: the sum is a whole number; a logarithm and its rounding are left)
    for got in (log_p, -entropy, top_p[:, 0]):
        assert ((got.double() - want).abs() <= 2.0 ** -24 * 8 * (1 + want.abs())).all(), (got[:6], want[:6])
    assert torch.equal(top_id[:, 0].long(), (x > -inf).int().argmax(1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=lambda d: NAME[d])
@ROWS
@pytest.mark.parametrize("shift", [0, 1, 3, 7])
@pytest.mark.parametrize("value", [3e9, -3e9, 1e30, 7e4])
def test_large_logits_among_masked_ones(value, rows, shift, dtype):
    """Equal logits of any size among -inf: one in front of the first 16-byte boundary, the others in the pieces of the same lane."""
    i = torch.arange(VOCAB)
    per = 16 // (torch.finfo(dtype).bits // 8)
    first = (per - shift % per) % per                         # values in front of the boundary
    places = [[0], [first + 255 * per], [first + 511 * per], [8000]]
    kinds = [torch.where(sum((i == p) for ps in places[:n] for p in ps).bool(), value, -float("inf")) for n in (1, 2, 3, 4)]
    x = _rows(kinds, rows, dtype, shift)
    from metalhlo_amd import kernels
    count = (x > -float("inf")).sum(1)
    log_p, entropy, top_p, top_id = kernels.token_log_probs(x, torch.zeros(rows, dtype=torch.int32, device="cuda"), top=1)
    want = -count.double().log()
    for got in (log_p, -entropy, top_p[:, 0]):
        assert ((got.double() - want).abs() <= 2.0 ** -24 * 8 * (1 + want.abs())).all(), (got[:6], want[:6])
    assert (top_id == 0).all()
